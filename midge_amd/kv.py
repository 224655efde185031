"""Paged k/v caches: batches of sequences, f16 or MXFP4 (mh_kv_*).

    append_dev(cache, batch, rows)     new rows of q, k, v: biases, norms of q
                                       and k, rotation, k and v into the cache
    attention_dev(cache, batch, ...)   attention over the cached tokens
    read_dev(cache, batch, k, v)       the stored values as f32
    check(cache, batch)                a batch in host memory, without a device

Trees of drafted tokens (parent: of each row the row that it follows, -1 for
the last cached token; at most 64 rows a sequence):

    tree_append_dev, tree_attention_dev, tree_check    the same for trees
    keep_dev(caches, batch, n_kept, kept, len_out)     the kept rows of all
                                       layers move up behind the cached tokens

The batched form of attention() (engine/midge.c:341-400) around its
projections. Pointers are device addresses (int, DevBuf) unless noted.
"""
from __future__ import annotations

import ctypes as C

from . import _lib
from ._lib import KV_F16, KV_MXFP4
from .device import DevBuf

__all__ = ["KV_F16", "KV_MXFP4", "KVCache", "KVBatch", "KVRows", "append_dev", "read_dev", "attention_ws", "attention_dev",
           "check", "tree_append_dev", "tree_attention_ws", "tree_attention_dev", "tree_check", "keep_dev"]


def _p(a) -> int:
    return int(a) if a is not None else 0


class KVCache:
    """A layer's pages: k, v [n_pages][n_kv_heads][page][head_dim] as f16 or
    MXFP4 codes, ks, vs the MXFP4 exponent bytes (of 32 elements each)."""

    def __init__(self, dt: int, n_kv_heads: int, head_dim: int, page: int, n_pages: int, k, v, ks=None, vs=None):
        self.c = _lib.MhKvCache(dt, n_kv_heads, head_dim, page, n_pages, _p(k), _p(v), _p(ks), _p(vs))
        self._bufs: list[DevBuf] = []

    @classmethod
    def alloc(cls, dt: int, n_kv_heads: int, head_dim: int, page: int, n_pages: int) -> "KVCache":
        """A cache in memory of its own (free() gives it back)."""
        n = n_pages * n_kv_heads * page * head_dim
        sizes = [2 * n] * 2 if dt == KV_F16 else [n // 2] * 2 + [n // 32] * 2
        bufs: list[DevBuf] = []
        try:
            for s in sizes:
                bufs.append(DevBuf(s))
        except Exception:       # (no room for a later one: those before it go back)
            for b in bufs:
                b.free()
            raise
        c = cls(dt, n_kv_heads, head_dim, page, n_pages, *bufs)
        c._bufs = bufs
        return c

    def free(self) -> None:
        """Gives alloc()'s memory back; the cache names none afterwards."""
        for b in self._bufs:
            b.free()
        if self._bufs:
            self.c.k = self.c.v = self.c.ks = self.c.vs = None
        self._bufs = []


class KVBatch:
    """The sequences of a call: rows row0[s] .. row0[s + 1] - 1 are the newest
    of sequence s's len[s] tokens (row0 0: one row each), pages[s][max_pages]
    its pages."""

    def __init__(self, n_seqs: int, n_rows: int, max_rows: int, max_pages: int, row0, len, pages):
        self.c = _lib.MhKvBatch(n_seqs, n_rows, max_rows, max_pages, _p(row0), _p(len), _p(pages))


class KVRows:
    """New rows of q, k and v, as the projections leave them."""

    def __init__(self, n_heads: int, ctx: int, norm_eps: float, q, k, v, ldq: int, ldk: int, ldv: int, q_out,
                 bq=None, bk=None, bv=None, qn=None, kn=None, rope_cos=None, rope_sin=None):
        self.c = _lib.MhKvRows(n_heads, ctx, norm_eps, _p(q), _p(k), _p(v), ldq, ldk, ldv, _p(q_out), _p(bq), _p(bk), _p(bv),
                               _p(qn), _p(kn), _p(rope_cos), _p(rope_sin))


def append_dev(cache: KVCache, batch: KVBatch, rows: KVRows) -> None:
    _lib.call("mh_kv_append_dev", C.byref(cache.c), C.byref(batch.c), C.byref(rows.c))


def read_dev(cache: KVCache, batch: KVBatch, k, v) -> None:
    _lib.call("mh_kv_read_dev", C.byref(cache.c), C.byref(batch.c), _p(k), _p(v))


def attention_ws(cache: KVCache, batch: KVBatch, n_heads: int) -> int:
    """Workspace bytes of attention_dev for this batch's sizes."""
    b = C.c_uint64()
    _lib.call("mh_kv_attention_ws", C.byref(cache.c), C.byref(batch.c), int(n_heads), C.byref(b))
    return int(b.value)


def attention_dev(cache: KVCache, batch: KVBatch, n_heads: int, q, out, ws, ws_bytes: int, scale: float, window: int = 0,
                  sink=None) -> None:
    _lib.call("mh_kv_attention_dev", C.byref(cache.c), C.byref(batch.c), int(n_heads), int(window), float(scale), _p(sink),
              _p(q), _p(out), _p(ws), int(ws_bytes))


def check(cache: KVCache, batch: KVBatch) -> None:
    """mh_kv_check: row0, len and pages of `batch` are HOST addresses here
    (without a window: every page up to a sequence's length counts)."""
    _lib.call("mh_kv_check", C.byref(cache.c), C.byref(batch.c))


def tree_append_dev(cache: KVCache, batch: KVBatch, parent, rows: KVRows) -> None:
    _lib.call("mh_kv_tree_append_dev", C.byref(cache.c), C.byref(batch.c), _p(parent), C.byref(rows.c))


def tree_attention_ws(cache: KVCache, batch: KVBatch, n_heads: int) -> int:
    """Workspace bytes of tree_attention_dev for this batch's sizes."""
    b = C.c_uint64()
    _lib.call("mh_kv_tree_attention_ws", C.byref(cache.c), C.byref(batch.c), int(n_heads), C.byref(b))
    return int(b.value)


def tree_attention_dev(cache: KVCache, batch: KVBatch, parent, n_heads: int, q, out, ws, ws_bytes: int, scale: float,
                       window: int = 0, sink=None) -> None:
    _lib.call("mh_kv_tree_attention_dev", C.byref(cache.c), C.byref(batch.c), _p(parent), int(n_heads), int(window), float(scale),
              _p(sink), _p(q), _p(out), _p(ws), int(ws_bytes))


def tree_check(cache: KVCache, batch: KVBatch, parent) -> None:
    """mh_kv_tree_check: row0, len and pages of `batch`, and parent, are HOST addresses."""
    _lib.call("mh_kv_tree_check", C.byref(cache.c), C.byref(batch.c), _p(parent))


def keep_dev(caches, batch: KVBatch, n_kept, kept, len_out) -> None:
    """Rows kept[s][:n_kept[s]] of each sequence's tree move to the slots
    behind its cached tokens in every cache of `caches` (KVCache each, the
    layers'); len_out[s] is the length then."""
    n = len(caches)     # (one copy: setting an array's structures one by one takes 13 us for 36 layers, this 3)
    a = (_lib.MhKvCache * n).from_buffer_copy(b"".join([c.c for c in caches])) if n else None
    _lib.call("mh_kv_keep_dev", a, n, C.byref(batch.c), _p(n_kept), _p(kept), _p(len_out))
