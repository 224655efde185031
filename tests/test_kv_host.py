"""Paged k/v caches and log probabilities without a GPU: refused arguments,
mh_kv_check on host batches, and the encoder that the tests compare with."""
import ctypes as C

import numpy as np
import pytest

from midge_amd import _lib
from midge_amd.kv import KV_F16, KV_MXFP4, KVBatch, KVCache, KVRows, check
from kv_oracle import LEVELS, decode, encode

ARG, DTYPE, RANGE, UNSUP, NOINIT = _lib.MH_E_ARG, _lib.MH_E_DTYPE, _lib.MH_E_RANGE, _lib.MH_E_UNSUPPORTED, _lib.MH_E_NOINIT
A = 4096    # an aligned address that nothing follows


def cache(**kw):
    c = dict(dt=KV_MXFP4, n_kv_heads=2, head_dim=64, page=16, n_pages=9, k=A, v=A, ks=A, vs=A)
    return KVCache(**{**c, **kw})


def batch(**kw):
    b = dict(n_seqs=2, n_rows=5, max_rows=4, max_pages=3, row0=A, len=A, pages=A)
    return KVBatch(**{**b, **kw})


def rows(**kw):
    r = dict(n_heads=4, ctx=99, norm_eps=1e-5, q=A, k=2 * A, v=3 * A, ldq=256, ldk=128, ldv=128, q_out=1 << 20, rope_cos=A, rope_sin=A)
    return KVRows(**{**r, **kw})


def rc(name, *a):
    return getattr(_lib.load(), name)(*a)


def append(c=None, b=None, r=None):
    return rc("mh_kv_append_dev", C.byref((c or cache()).c), C.byref((b or batch()).c), C.byref((r or rows()).c))


def attend(c=None, b=None, nh=4, window=0, scale=0.125, q=A, out=1 << 20, ws=1 << 32, n=1 << 40):
    return rc("mh_kv_attention_dev", C.byref((c or cache()).c), C.byref((b or batch()).c), nh, window, scale, None, q, out, ws, n)


@pytest.mark.parametrize("kw,code", [
    (dict(dt=2), DTYPE), (dict(head_dim=48), UNSUP), (dict(head_dim=0), ARG), (dict(n_kv_heads=0), ARG), (dict(page=8), ARG),
    (dict(page=48), ARG), (dict(page=8192), ARG), (dict(n_pages=0), ARG), (dict(n_pages=1 << 31), ARG), (dict(k=0), ARG),
    (dict(ks=0), ARG), (dict(v=A + 8), ARG), (dict(vs=A + 1), ARG)])
def test_cache_refusals(kw, code):
    c = cache(**kw)
    assert append(c=c) == code and attend(c=c) == code
    assert rc("mh_kv_read_dev", C.byref(c.c), C.byref(batch().c), A, None) == code
    assert rc("mh_kv_attention_ws", C.byref(c.c), C.byref(batch().c), 4, C.byref(C.c_uint64())) == code


@pytest.mark.parametrize("kw", [
    dict(n_seqs=0), dict(n_rows=-1), dict(max_rows=0), dict(max_pages=0), dict(max_pages=1 << 28), dict(len=0), dict(pages=0),
    dict(row0=0), dict(len=A + 2), dict(n_rows=1 << 24)])
def test_batch_refusals(kw):
    b = batch(**kw)
    assert append(b=b) == ARG and attend(b=b) == ARG
    assert rc("mh_kv_read_dev", C.byref(cache().c), C.byref(b.c), A, None) == ARG


@pytest.mark.parametrize("kw", [
    dict(n_heads=0), dict(n_heads=3), dict(ldq=255), dict(ldk=127), dict(ldv=0), dict(q=0), dict(v=0), dict(q_out=0), dict(rope_sin=0),
    dict(ctx=0), dict(q=A + 2), dict(norm_eps=-1.0, qn=A), dict(norm_eps=float("nan"), kn=A),
    dict(q_out=A + 4), dict(ldq=512, q_out=A), dict(q_out=2 * A), dict(q_out=3 * A + 64)])
def test_append_refusals(kw):
    assert append(r=rows(**kw)) == ARG


def test_attention_refusals():
    for kw in (dict(nh=3), dict(nh=0), dict(window=-1), dict(scale=float("nan")), dict(scale=float("inf")), dict(q=0), dict(out=0),
               dict(ws=0), dict(ws=A + 8), dict(n=0), dict(out=A + 4), dict(q=A + 1), dict(q=A + 4), dict(out=(1 << 20) + 8), dict(scale=3e38),
               dict(ws=A), dict(ws=(1 << 20) + 256)):
        assert attend(**kw) == ARG, kw
    lib = _lib.load()
    for args in ((None, C.byref(batch().c)), (C.byref(cache().c), None)):
        assert lib.mh_kv_attention_dev(*args, 4, 0, 1.0, None, A, 1 << 20, 1 << 32, 1 << 40) == ARG
        assert lib.mh_kv_append_dev(*args, C.byref(rows().c)) == ARG and lib.mh_kv_read_dev(*args, A, None) == ARG
    assert lib.mh_kv_append_dev(C.byref(cache().c), C.byref(batch().c), None) == ARG
    assert lib.mh_kv_attention_ws(C.byref(cache().c), C.byref(batch().c), 4, None) == ARG
    assert rc("mh_kv_read_dev", C.byref(cache().c), C.byref(batch().c), None, None) == ARG
    assert rc("mh_kv_read_dev", C.byref(cache().c), C.byref(batch().c), A, A + 4) == ARG


def test_units_that_the_counts_hold():
    """Sequences x heads past a grid, or so many pages that the work units pass 2^41."""
    far = dict(out=1 << 56, ws=1 << 58, n=1 << 60)
    assert attend(c=cache(n_kv_heads=1024), b=batch(n_seqs=1 << 20, n_rows=1 << 20, max_rows=1), nh=1024, **far) == UNSUP
    assert attend(c=cache(n_kv_heads=16), b=batch(n_seqs=1 << 20, n_rows=1 << 20, max_rows=1), nh=16, **far) == UNSUP
    assert attend(c=cache(page=4096), b=batch(n_seqs=64, max_pages=1 << 18), **far) == UNSUP
    assert attend(c=cache(n_kv_heads=1024, page=4096), b=batch(n_seqs=1 << 20, n_rows=1 << 20, max_rows=1, max_pages=1 << 18), nh=1024, **far) == UNSUP


def logprobs(**kw):
    a = dict(logits=A, ld=100, n=2, V=100, ids=A, m=1, top=5, lp=A, ent=A, ti=A, tl=A, ws=A, nb=1 << 40)
    a.update(kw)
    return rc("mh_logprobs_dev", *a.values())


def test_logprobs_refusals():
    for kw in (dict(logits=0), dict(ld=99), dict(n=-1), dict(n=1 << 24), dict(V=0), dict(V=(1 << 30) + 1, ld=1 << 31), dict(m=-1), dict(ids=0), dict(lp=0),
               dict(top=65), dict(top=-1), dict(top=5, V=4), dict(ti=0), dict(tl=0), dict(ws=0), dict(nb=0), dict(ws=A + 8),
               dict(logits=A + 2), dict(m=0, top=0, ent=0)):
        assert logprobs(**kw) == ARG, kw
    assert rc("mh_logprobs_ws", 1, 100, 101, C.byref(C.c_uint64())) == ARG and rc("mh_logprobs_ws", 1, 100, 5, None) == ARG


def test_calls_before_init():
    if _lib.load().mh_sync() != NOINIT:
        pytest.skip("the library is initialised")
    assert append() == NOINIT and attend() == NOINIT and logprobs() == NOINIT


def host(seqs, table, n_rows=6, max_rows=4, **kw):
    row0 = np.array([0] + list(np.cumsum([r for _, r in seqs])), np.int32)
    ln = np.array([n for n, _ in seqs], np.int32)
    pages = np.array(table, np.int32)
    b = KVBatch(len(seqs), n_rows, max_rows, pages.shape[1], row0.ctypes.data, ln.ctypes.data, pages.ctypes.data)
    b.keep = row0, ln, pages
    for k, v in kw.items():
        {"row0": row0, "len": ln, "pages": pages}[k].__setitem__(*v)
    return b


GOOD = ([(33, 2), (0, 0), (16, 4)], [[8, 0, 3], [-1, -1, -1], [5, -1, -1]])


@pytest.mark.parametrize("kw,bad", [
    ({}, None), (dict(row0=(3, 7)), 2), (dict(row0=(1, 5)), 0), (dict(row0=(0, -1)), 0), (dict(row0=(2, 1)), 1), (dict(len=(0, 49)), 0),
    (dict(len=(2, -1)), 2), (dict(len=(2, 17)), 2), (dict(pages=((0, 2), 9)), 0), (dict(pages=((0, 0), -1)), 0),
    (dict(pages=((0, 1), 1 << 30)), 0)])
def test_check(kw, bad):
    c, b = cache(), host(*GOOD, **kw)
    if bad is None:
        check(c, b)
        return
    with pytest.raises(_lib.MidgeHipError, match=f"sequence {bad}:") as e:
        check(c, b)
    assert e.value.code == RANGE


def test_check_without_row0():
    ln, pages = np.array([3, 17], np.int32), np.array([[1, -1], [2, 3]], np.int32)
    b = KVBatch(2, 2, 1, 2, 0, ln.ctypes.data, pages.ctypes.data)
    check(cache(), b)
    pages[1, 1] = 9
    with pytest.raises(_lib.MidgeHipError, match="sequence 1:"):
        check(cache(), b)


def test_encoder_definition():
    """encode() holds what the header says: the smallest exponent, the nearest code, ties to even, NaN blocks."""
    rng = np.random.default_rng(0)
    x = (rng.standard_normal((2000, 32)) * 2.0 ** rng.integers(-16, 16, (2000, 1))).astype(np.float32)
    x[0], x[1, 3], x[2, 5] = 0, np.inf, np.nan
    codes, e = encode(x)
    d = decode(codes, e)
    assert e[1] == 255 and e[2] == 255 and np.isnan(d[1:3]).all() and (d[0] == 0).all() and e[0] == 114
    ok = e[:, 0] != 255
    top, s = np.abs(x[ok]).max(-1).astype(np.float64), 2.0 ** (e[ok, 0].astype(np.float64) - 127)
    assert ((top <= 7 * s) | (s == 2.0 ** 13)).all() and ((top > 7 * s / 2) | (s == 2.0 ** -13)).all()
    grid = np.concatenate((LEVELS, -LEVELS))
    best = np.abs(x[ok].astype(np.float64)[..., None] - grid * s[:, None, None]).min(-1)
    assert (np.abs(d[ok] - x[ok]) == best).all()
    ties = np.zeros((1, 32), np.float32)
    ties[0, :8] = [6, 0.25, 0.75, 1.25, -1.75, 2.5, 3.5, 5]
    assert (decode(*encode(ties))[0, :8] == [6, 0, 1, 1, -2, 2, 4, 4]).all()


# -------------------------------------------------- workspaces of a server

def lp_ws(n, V, top):
    b = C.c_uint64()
    assert rc("mh_logprobs_ws", n, V, top, C.byref(b)) == 0
    return b.value


@pytest.mark.parametrize("V", [1, 100, 1023, 1024, 1025, 4096, 5000, 32000, 50257, 131072, 201088, 600000, 1 << 20, 1 << 22])
def test_logprobs_workspace_of_the_largest_call(V):
    """A workspace for some rows, tokens and alternatives serves every smaller call: its size never falls as they grow,
    also where a call is cut in another way."""
    ns = sorted({*range(1, 80), *(n + d for n in (128, 256, 400, 511, 1024, 2048, 4096, 10000, 1 << 20) for d in (-1, 0, 1)),
                 *((1 << 20) // V + d for d in (-1, 0, 1, 2)), (1 << 24) - 1} - {0, -1})
    for top in (0, min(20, V)):
        sizes = [lp_ws(n, V, top) for n in ns]
        assert all(a <= b for a, b in zip(sizes, sizes[1:])), [(n, a, b) for n, a, b in zip(ns, sizes, sizes[1:]) if a > b][:3]
        assert all(lp_ws(n, v, top) <= s for n, s in list(zip(ns, sizes))[::7] for v in (V - 1, V // 2, V * 3 // 4, V // 5) if v >= max(top, 1))
    if V >= 64:
        assert all(lp_ws(n, V, t) < lp_ws(n, V, t + 1) for n in (1, 33, 500) for t in range(64))


@pytest.mark.parametrize("V", [1000, 32000, 201088])
def test_logprobs_calls_on_a_larger_workspace(V):
    """The workspace of n rows is enough for every call of fewer."""
    if _lib.load().mh_sync() != NOINIT:
        pytest.skip("the library is initialised")
    for n in (6, 21, 33, 400, 2000):
        for k in [*range(1, 40), 200, 1040]:
            if k <= n:
                assert logprobs(n=k, V=V, ld=V, top=20, nb=lp_ws(n, V, 20)) == NOINIT, (n, k)
    assert logprobs(n=3, V=V, ld=V, top=20, nb=16 + 3 * 176 - 1) == ARG


@pytest.mark.parametrize("dt", [KV_F16, KV_MXFP4])
@pytest.mark.parametrize("hd,nkv,group", [(64, 8, 8), (128, 4, 8), (128, 8, 4), (256, 1, 8), (256, 2, 16), (32, 3, 5), (96, 1, 64)])
def test_attention_workspace_of_the_largest_batch(dt, hd, nkv, group):
    """A workspace for the most sequences, rows and rows a sequence serves every smaller batch of the cache."""
    c = cache(dt=dt, head_dim=hd, n_kv_heads=nkv)

    def ws(seqs, rows, most, row0=A):
        size = C.c_uint64()
        assert rc("mh_kv_attention_ws", C.byref(c.c), C.byref(batch(n_seqs=seqs, n_rows=rows, max_rows=most, row0=row0).c), nkv * group,
                  C.byref(size)) == 0
        return size.value
    seqs, mosts = [1, 2, 3, 7, 8, 31, 64, 255, 256, 257, 1000], [1, 2, 3, 4, 5, 6, 7, 8, 9, 12, 16, 17, 33, 64, 100, 512]
    for i, s in enumerate(seqs):
        for rows in (s, s + 5, 64, 513, 5000):
            sizes = [ws(s, rows, m) for m in mosts]
            assert all(a <= b for a, b in zip(sizes, sizes[1:])), (s, rows)
            for m, size in zip(mosts, sizes):
                assert ws(s, rows + 1, m) >= size and (i == 0 or ws(seqs[i - 1], rows, m) <= size)
                assert rows != s or ws(s, s, 1, 0) <= size


# ---------------------------------------------------- weights under outputs

def test_weights_under_outputs_are_refused():
    """q_out over a bias, norm weight or rotation table, and out or the workspace over the sinks, by as little as a float."""
    o = 1 << 20             # q_out: 5 rows of 4 heads of 64
    size = 5 * 256 * 4
    for name, n in (("bq", 256), ("bk", 128), ("bv", 128), ("qn", 64), ("kn", 64), ("rope_cos", 99 * 32), ("rope_sin", 99 * 32)):
        for at in (o, o + size - 4, o + 4 - 4 * n):
            assert append(r=rows(**{name: at})) == ARG, (name, at - o)
    assert rc("mh_kv_append_dev", C.byref(cache().c), C.byref(batch(n_rows=0).c), C.byref(rows(bq=o).c)) in (0, NOINIT)      # no row, no output

    def with_sink(at):
        return rc("mh_kv_attention_dev", C.byref(cache().c), C.byref(batch().c), 4, 0, 0.125, at, A, o, 1 << 32, 1 << 40)
    need = C.c_uint64()
    assert rc("mh_kv_attention_ws", C.byref(cache().c), C.byref(batch().c), 4, C.byref(need)) == 0
    for at in (o, o + size - 4, o - 12, 1 << 32, (1 << 32) + need.value - 4, (1 << 32) - 12):
        assert with_sink(at) == ARG, at
    if _lib.load().mh_sync() == NOINIT:
        for at in (o + size, o - 16, (1 << 32) + need.value, A):
            assert with_sink(at) == NOINIT, at
        for name, n in (("bq", 256), ("kn", 64), ("rope_sin", 99 * 32)):
            assert append(r=rows(**{name: o + size})) == NOINIT and append(r=rows(**{name: o - 4 * n})) == NOINIT


# ------------------------------------------------- memory of a cache's own

class FakeBuf:
    live: list = []

    def __init__(self, nbytes):
        if len(FakeBuf.live) == FakeBuf.room:
            raise _lib.MidgeHipError(_lib.MH_E_NOMEM, "mh_alloc", "full")
        self.ptr, self.nbytes = 4096 * (len(FakeBuf.live) + 1), nbytes
        FakeBuf.live.append(self)

    def __int__(self):
        return self.ptr

    def free(self):
        if self.ptr:
            FakeBuf.live.remove(self)
            self.ptr = 0


@pytest.mark.parametrize("dt,arrays", [(KV_F16, 2), (KV_MXFP4, 4)])
def test_alloc_that_does_not_fit(monkeypatch, dt, arrays):
    """A cache whose second or later array has no room gives back those before it."""
    from midge_amd import kv
    monkeypatch.setattr(kv, "DevBuf", FakeBuf)
    FakeBuf.live = []
    for FakeBuf.room in range(arrays):
        with pytest.raises(_lib.MidgeHipError):
            KVCache.alloc(dt, 2, 64, 16, 9)
        assert not FakeBuf.live
    FakeBuf.room = arrays
    c = KVCache.alloc(dt, 2, 64, 16, 9)
    n = 9 * 2 * 16 * 64
    assert [b.nbytes for b in FakeBuf.live] == ([2 * n] * 2 if dt == KV_F16 else [n // 2] * 2 + [n // 32] * 2)
    c.free()
    assert not FakeBuf.live


def test_freed_cache_is_refused(monkeypatch):
    """A cache given back names no memory: calls on it are refused, whoever has the addresses now."""
    from midge_amd import kv
    monkeypatch.setattr(kv, "DevBuf", FakeBuf)
    FakeBuf.live, FakeBuf.room = [], 4
    c = KVCache.alloc(KV_MXFP4, 2, 64, 16, 9)
    c.free()
    c.free()
    assert append(c=c) == ARG and attend(c=c) == ARG and rc("mh_kv_read_dev", C.byref(c.c), C.byref(batch().c), A, None) == ARG
    mine = cache()      # the caller's own memory stays the caller's
    mine.free()
    assert mine.c.k == A and mine.c.vs == A


def test_misaligned_weights_are_refused():
    """Biases, norm weights, tables and sinks off a 4-byte address, as rows are."""
    for name in ("bq", "bk", "bv", "qn", "kn", "rope_cos", "rope_sin"):
        for off in (1, 2):
            assert append(r=rows(**{name: A + off})) == ARG, name
    for off in (1, 2):
        assert rc("mh_kv_attention_dev", C.byref(cache().c), C.byref(batch().c), 4, 0, 0.125, A + off, A, 1 << 20, 1 << 32, 1 << 40) == ARG
