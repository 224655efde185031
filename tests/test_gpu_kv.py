"""Paged k/v caches on the GPU: the append, the read-back and the attention
against their definition in 64 bits (kv_oracle), over cache types, head
layouts, page sizes, ragged batches, masks and what stale slots may hold."""
import contextlib

import numpy as np
import pytest

from conftest import say
from midge_amd import DevBuf, MidgeHipError, sync
from midge_amd import kv
from hip_graph import Graph, Stream
from kv_oracle import KV_F16, KV_MXFP4, Batch, KVRows, Pages, attention, decode, encode, f16, prepared

pytestmark = pytest.mark.gpu

F32 = np.float32
EPS = 1e-5


def tables(ctx, hd):
    ang = np.arange(ctx)[:, None] * 10000.0 ** (-np.arange(hd // 2) / (hd // 2))
    return np.cos(ang).astype(F32), np.sin(ang).astype(F32)


class Dev:
    """Device copies, freed together."""

    def __init__(self):
        self.bufs = []

    def __call__(self, a):
        b = DevBuf.from_array(np.ascontiguousarray(a))
        self.bufs.append(b)
        return b

    def free(self, *more):
        for b in [*self.bufs, *more]:
            b.free()


# ------------------------------------------------------------------ append

APPEND = [
    # dt, nh, nkv, hd, page, seqs [(len, rows)], norm, bias, rope, fused, extra rows
    (KV_MXFP4, 64, 8, 64, 64, [(1, 1)], 0, 1, 1, 0, 0),
    (KV_MXFP4, 64, 8, 64, 16, [(17, 17), (40, 3), (16, 1)], 0, 1, 1, 1, 2),
    (KV_F16, 32, 4, 128, 16, [(9, 1), (33, 1), (16, 1)], 1, 0, 1, 0, 0),
    (KV_MXFP4, 4, 4, 32, 32, [(70, 35), (0, 0), (2, 5)], 1, 1, 1, 1, 1),
    (KV_F16, 6, 2, 96, 128, [(200, 129)], 1, 1, 1, 1, 0),
    (KV_MXFP4, 6, 2, 96, 16, [(19, 7)], 0, 0, 1, 0, 0),
    (KV_MXFP4, 3, 1, 192, 64, [(65, 3), (64, 64)], 1, 0, 0, 1, 3),
    (KV_MXFP4, 8, 1, 256, 256, [(300, 47), (0, 2)], 1, 1, 1, 0, 0),
    (KV_F16, 8, 8, 64, 32, [(33, 33)], 0, 0, 0, 0, 0),
]


@pytest.mark.parametrize("dt,nh,nkv,hd,page,seqs,norm,bias,rope,fused,extra", APPEND)
def test_append(mh, dt, nh, nkv, hd, page, seqs, norm, bias, rope, fused, extra):
    say(f"kv append dt={dt} heads={nh}/{nkv}x{hd} page={page} seqs={seqs} norm={norm} bias={bias} rope={rope} fused={fused}")
    rng = np.random.default_rng(nh * hd + page)
    pg, b, dev = None, Batch(seqs, page, rng, extra), Dev()
    pg = Pages(dt, nkv, hd, page, b.n_pages, rng)
    n, (wq, wk) = b.n_rows, (nh * hd, nkv * hd)
    pad = 5 if fused else 0     # a row stride that keeps no row 16-byte aligned
    m = rng.standard_normal((n, wq + 2 * wk + pad)).astype(F32)
    q, k, v = m[:, :wq], m[:, wq:wq + wk], m[:, wq + wk:wq + 2 * wk]
    bq, bk, bv = [rng.standard_normal(w).astype(F32) if bias else None for w in (wq, wk, wk)]
    qn, kn = [(1 + 0.1 * rng.standard_normal(hd)).astype(F32) if norm else None for _ in "qk"]
    ctx = max(x for x, _ in seqs) + 1
    co, si = tables(ctx, hd) if rope else (None, None)
    ptr = lambda a: dev(a).ptr if a is not None else 0     # noqa: E731
    qo = dev(np.full((n, wq), 7.5, F32))
    if fused:
        at, ld = ptr(m), [m.shape[1]] * 3
        src = [at, at + 4 * wq, at + 4 * (wq + wk)]
    else:
        src, ld = [ptr(a) for a in (q, k, v)], [wq, wk, wk]
    r = KVRows(nh, ctx, EPS, *src, *ld, qo, ptr(bq), ptr(bk), ptr(bv), ptr(qn), ptr(kn), ptr(co), ptr(si))
    kv.append_dev(pg.cache, b.batch, r)
    ko, vo = dev(np.full((n, wk), 7.5, F32)), dev(np.full((n, wk), 7.5, F32))
    kv.read_dev(pg.cache, b.batch, ko, vo)
    sync()
    want_q, want_kv = np.full((n, wq), 7.5), [np.full((n, wk), 7.5), np.full((n, wk), 7.5)]
    for row, s, pos in b.rows():
        if pos < 0:
            continue
        c, sn = (co[pos], si[pos]) if rope else (None, None)
        want_q[row] = prepared(q[row].reshape(nh, hd), bq, qn, EPS, c, sn).ravel()
        pair = [prepared(k[row].reshape(nkv, hd), bk, kn, EPS, c, sn).astype(F32), prepared(v[row].reshape(nkv, hd), bv, None, EPS, None, None).astype(F32)]
        for w, x in enumerate(pair):
            pg.put(b.pages[s], pos, w, x)
            want_kv[w][row] = (f16(x).astype(np.float64) if dt == KV_F16 else decode(*encode(x))).ravel()
    got = pg.download()
    for a, g in zip(pg.arr, got):       # every other slot as it was, too
        assert (a == g).all(), (a != g).sum()
    # one rounding of the 64-bit value
    gq = qo.download(F32, (n, wq)).astype(np.float64)
    assert (np.abs(gq - want_q) <= 2.0 ** -24 * np.abs(want_q) + 1e-38).all()
    for w, o in enumerate((ko, vo)):
        assert (o.download(F32, (n, wk)) == want_kv[w]).all()
    # one of the two alone, the other left out
    kv.read_dev(pg.cache, b.batch, None, ko)
    sync()
    assert (ko.download(F32, (n, wk)) == want_kv[1]).all()
    dev.free(pg, b)


@pytest.mark.parametrize("dt", [KV_F16, KV_MXFP4])
def test_append_special_values(mh, dt):
    """Infinities, NaN, zeros of both signs, subnormals, ties and magnitudes past the type's."""
    say(f"kv append special values dt={dt}")
    rng, hd = np.random.default_rng(3), 64
    x = rng.standard_normal((8, hd)).astype(F32)
    x[0, 3], x[1, 40], x[2] = np.inf, np.nan, 0.0
    x[3], x[3, 0] = np.float32(1e-40), -0.0
    x[4, :32] = [6, 0.25, 0.75, 1.25, -1.75, 2.5, -3.5, 5] * 4
    x[4, 32:] = [7, 0.25, 0.75, 1.25, -1.75, 2.5, -3.5, np.nextafter(F32(5), F32(6))] * 4
    x[5] *= 1e5
    x[6] *= np.float32(2.0 ** -16)
    x[7, :4] = [65519, 65520, -65536, 2.0 ** -14]
    b, dev = Batch([(8, 8)], 16, rng), Dev()
    pg = Pages(dt, 1, hd, 16, b.n_pages, rng)
    d, qo = dev(x), dev(np.zeros((8, hd), F32))
    kv.append_dev(pg.cache, b.batch, KVRows(1, 1, 0.0, d, d, d, hd, hd, hd, qo))
    sync()
    for t in range(8):
        for w in (0, 1):
            pg.put(b.pages[0], t, w, x[t][None])
    got = pg.download()
    for i, (a, g) in enumerate(zip(pg.arr, got)):
        if dt == KV_MXFP4 and i < 2:        # the codes of a NaN block say nothing
            for t in range(8):
                at = (b.pages[0][0], 0, t)
                live = np.repeat(pg.arr[i + 2][at] != 255, 16)
                assert (a[at][live] == g[at][live]).all(), (i, t)
        elif dt == KV_F16:
            av, gv = a.view(np.float16), g.view(np.float16)
            assert ((a == g) | (np.isnan(av) & np.isnan(gv))).all()
        else:
            assert (a == g).all()
    assert np.array_equal(qo.download(F32, (8, hd)), x, equal_nan=True)
    dev.free(pg, b)


def test_append_in_place_q_and_rope_bounds(mh):
    """q_out may be q; a row past the tables is not stored, and mh_sync says so."""
    say("kv append in place, positions past the tables")
    rng, hd = np.random.default_rng(5), 64
    b, dev = Batch([(20, 4)], 16, rng), Dev()
    pg = Pages(KV_F16, 2, hd, 16, b.n_pages, rng)
    co, si = tables(18, hd)       # positions 16, 17 of 16..19
    q, k, v = [rng.standard_normal((4, w * hd)).astype(F32) for w in (4, 2, 2)]
    dq = dev(q)
    kv.append_dev(pg.cache, b.batch, KVRows(4, 18, EPS, dq, dev(k), dev(v), 4 * hd, 2 * hd, 2 * hd, dq, rope_cos=dev(co), rope_sin=dev(si)))
    with pytest.raises(MidgeHipError, match="out of bounds"):
        sync()
    sync()      # said once
    want = q.astype(np.float64)
    for row, s, pos in b.rows():
        if pos < 18:
            want[row] = prepared(q[row].reshape(4, hd), None, None, EPS, co[pos], si[pos]).ravel()
            pg.put(b.pages[0], pos, 0, prepared(k[row].reshape(2, hd), None, None, EPS, co[pos], si[pos]).astype(F32))
            pg.put(b.pages[0], pos, 1, v[row].reshape(2, hd))
    assert (np.abs(dq.download(F32, q.shape) - want) <= 2.0 ** -24 * np.abs(want)).all()
    assert all((a == g).all() for a, g in zip(pg.arr, pg.download()))
    dev.free(pg, b)


# --------------------------------------------------------------- attention

def tolerance(mag, vmax, n):
    """Absolute error of an output: a score is off by two 22-bit terms' products
    and 32-bit sums (2^-21 of its terms' magnitudes), the weights by twice that
    and the exponential's and its argument's rounding (2^-22 each, and 2^-23 of
    the score), the weighted sum and the weights' sum by 2^-24 a step at most
    sqrt(n) of them (rounding to nearest), against values of at most vmax."""
    return (2 * 2.0 ** -21 * mag + 2.0 ** -22 * (4 + mag) + 2.0 ** -23 * np.sqrt(n)) * vmax


def run_attention(pg, b, nh, q, scale, window=0, sink=None, dev=None):
    """(out with 7.5 where nothing was written)"""
    own = dev or Dev()
    out = own(np.full((b.n_rows, nh * pg.hd), 7.5, F32))
    n = kv.attention_ws(pg.cache, b.batch, nh)
    ws = own(np.zeros(n, np.uint8))
    kv.attention_dev(pg.cache, b.batch, nh, own(q), out, ws, n, scale, window, own(sink) if sink is not None else None)
    sync()
    r = out.download(F32, (b.n_rows, nh * pg.hd))
    if dev is None:
        own.free()
    return r


def compare(pg, b, nh, q, scale, window, sink, got, rows=None):
    cache, worst = {}, 0.0
    seen = np.zeros(b.n_rows, bool)
    for row, s, pos in b.rows():
        seen[row] = True
        if rows is not None and row not in rows:
            continue
        if s not in cache:
            cache[s] = [pg.tokens(b.pages[s], b.seqs[s][0], w) for w in (0, 1)]
        k, v = cache[s]
        lo = max(0, pos + 1 - window) if window else 0
        k, v = k[:, lo:max(pos + 1, 0)], v[:, lo:max(pos + 1, 0)]
        want, mag = attention(q[row].reshape(nh, -1), k, v, scale, sink)
        vmax = np.abs(v).max() if v.size else 0.0
        err = np.abs(got[row].reshape(nh, -1) - want).max() if want.size else 0.0
        tol = tolerance(mag, vmax, max(pos + 1, 1))
        assert err <= tol, (row, s, pos, err, tol)
        worst = max(worst, err / tol if tol else 0.0)
    assert (got[~seen] == 7.5).all()
    return worst


ATTEND = [
    # dt, nh, nkv, hd, page, seqs [(len, rows)], window, sink, extra rows
    (KV_MXFP4, 64, 8, 64, 64, [(1, 1)], 0, 1, 0),
    (KV_MXFP4, 64, 8, 64, 16, [(17, 1), (300, 1), (0, 1), (64, 1), (65, 1), (1000, 1)], 0, 1, 2),
    (KV_F16, 64, 8, 64, 64, [(1025, 1), (256, 1), (257, 1)], 128, 0, 0),
    (KV_MXFP4, 32, 8, 128, 32, [(777, 1), (31, 1), (4000, 1)], 0, 0, 0),
    (KV_F16, 32, 4, 128, 16, [(500, 2), (90, 3), (2, 5), (0, 0), (33, 1)], 0, 1, 1),
    (KV_MXFP4, 32, 4, 128, 64, [(500, 4), (4, 4)], 100, 1, 0),
    (KV_MXFP4, 4, 4, 32, 256, [(700, 8), (3, 3)], 0, 0, 0),
    (KV_F16, 16, 16, 64, 128, [(333, 8)], 50, 1, 0),
    (KV_MXFP4, 6, 2, 96, 16, [(257, 1), (100, 5)], 0, 1, 0),
    (KV_F16, 24, 2, 96, 32, [(400, 3)], 0, 0, 0),
    (KV_MXFP4, 12, 4, 192, 64, [(200, 2)], 0, 0, 0),
    (KV_F16, 8, 1, 256, 16, [(129, 1), (64, 6)], 0, 1, 0),
    (KV_MXFP4, 8, 1, 256, 64, [(700, 1)], 0, 1, 0),
    (KV_F16, 40, 1, 64, 64, [(100, 1), (77, 2)], 0, 0, 0),
    # prompt chunks
    (KV_MXFP4, 64, 8, 64, 64, [(130, 130)], 0, 1, 0),
    (KV_MXFP4, 64, 8, 64, 16, [(200, 100), (33, 33), (1, 1), (0, 0), (500, 20)], 128, 1, 3),
    (KV_F16, 32, 8, 128, 128, [(300, 161)], 0, 0, 0),
    (KV_MXFP4, 32, 4, 128, 32, [(97, 97), (1200, 40)], 0, 1, 0),
    (KV_F16, 4, 4, 32, 16, [(290, 290)], 33, 0, 0),
    (KV_MXFP4, 6, 2, 96, 64, [(150, 120), (20, 30)], 0, 1, 0),
    (KV_F16, 6, 2, 96, 64, [(100, 70)], 0, 0, 0),
    (KV_MXFP4, 12, 4, 192, 64, [(140, 66)], 0, 0, 0),
    (KV_F16, 3, 1, 192, 64, [(120, 90)], 20, 1, 0),
    (KV_F16, 8, 1, 256, 16, [(129, 65)], 0, 1, 0),
    (KV_MXFP4, 8, 1, 256, 64, [(300, 33)], 7, 0, 0),
    (KV_MXFP4, 40, 1, 64, 64, [(222, 11)], 0, 0, 0),
    (KV_MXFP4, 4, 4, 32, 16, [(290, 290)], 33, 1, 0),
    (KV_F16, 8, 2, 64, 32, [(290, 150), (40, 33)], 0, 1, 0),
    # segments that more than one block takes, rows of nothing but padding, large pages
    (KV_MXFP4, 16, 2, 64, 1024, [(2500, 70), (10, 200), (700, 60)], 0, 1, 2),
    (KV_F16, 16, 2, 64, 4096, [(1900, 50)], 900, 0, 0),
    (KV_F16, 8, 1, 128, 64, [(1300, 60)], 0, 1, 0),
    (KV_MXFP4, 4, 1, 256, 64, [(900, 40)], 0, 0, 0),
    (KV_MXFP4, 64, 8, 64, 2048, [(5000, 1), (3, 1), (2100, 1)], 0, 1, 0),
]
# columns of one, two and four operands for every head width and type
ATTEND += [(dt, g * 2, 2, hd, 32, [(330, r), (70, 1), (5, r), (0, 1)], w, 1, 1)
           for dt in (KV_F16, KV_MXFP4) for hd in (32, 64, 96, 128, 192, 256) for g, r, w in ((1, 8, 0), (2, 5, 60), (4, 8, 0))]
ATTEND += [(dt, g * 2, 2, hd, 64, [(r, r), (700, 1), (90, r), (333, r - 2)], w, 1, 2)
           for dt in (KV_F16, KV_MXFP4) for hd in (32, 64, 96, 128, 192, 256) for g, r, w in ((8, 5, 0), (4, 16, 70), (13, 4, 0))]


@pytest.mark.parametrize("dt,nh,nkv,hd,page,seqs,window,sink,extra", ATTEND)
def test_attention(mh, dt, nh, nkv, hd, page, seqs, window, sink, extra):
    say(f"kv attention dt={dt} heads={nh}/{nkv}x{hd} page={page} seqs={seqs} window={window} sink={sink}")
    rng = np.random.default_rng(nh * hd + page + len(seqs))
    b = Batch(seqs, page, rng, extra, one=all(r == 1 for _, r in seqs) and not extra)
    pg = Pages(dt, nkv, hd, page, b.n_pages, rng)       # stale slots hold anything, NaN and inf among it
    for s, (n, _) in enumerate(seqs):
        pg.fill(b.pages[s], n, rng)
    pg.upload()
    q = (rng.standard_normal((b.n_rows, nh * hd)) * 1.5).astype(F32)
    sk = rng.standard_normal(nh).astype(F32) if sink else None
    scale = float(F32(hd ** -0.5))
    got = run_attention(pg, b, nh, q, scale, window, sk)
    worst = compare(pg, b, nh, q, scale, window, sk, got)
    say(f"  worst error {worst:.3f} of the tolerance")
    pg.free(), b.free()


@pytest.mark.parametrize("dt", [KV_F16, KV_MXFP4])
@pytest.mark.parametrize("rows", [1, 3, 70])
def test_attention_hard_scores(mh, dt, rows):
    """Large scores (one token takes all), tiny and large q and v, a negative and a zero scale, a window of one."""
    rng, nh, nkv, hd, n = np.random.default_rng(11), 16, 2, 64, 700
    for qs, vs, scale, window in ((30.0, 1.0, 0.125, 0), (1e-6, 1.0, 0.125, 0), (1.0, 1e-3, 0.125, 0), (1.0, 3e3, -0.3, 0), (1.0, 1.0, 0.0, 0),
                                  (1e4, 1.0, 1e-4, 0), (1.0, 1.0, 0.125, 1)):
        say(f"kv attention hard dt={dt} rows={rows} q*{qs} v*{vs} scale={scale} window={window}")
        b = Batch([(n, rows)], 64, rng)
        pg = Pages(dt, nkv, hd, 64, b.n_pages, rng)
        for w, std in ((0, 1.0), (1, vs)):
            for t in range(n):
                pg.put(b.pages[0], t, w, (rng.standard_normal((nkv, hd)) * std).astype(F32))
        pg.upload()
        q = (rng.standard_normal((b.n_rows, nh * hd)) * qs).astype(F32)
        got = run_attention(pg, b, nh, q, scale, window)
        compare(pg, b, nh, q, scale, window, None, got)
        pg.free(), b.free()


@pytest.mark.parametrize("dt", [KV_F16, KV_MXFP4])
@pytest.mark.parametrize("nh,nkv,hd,seqs,bad,window", [
    (8, 1, 64, (1500, 150), 1400, 0), (8, 1, 64, (2000, 5), 1998, 0), (8, 1, 64, (300, 4), 298, 0), (8, 1, 64, (300, 4), 290, 8), (4, 2, 128, (260, 200), 100, 0), (4, 2, 128, (260, 200), 100, 40),
    (64, 8, 64, (90, 90), 63, 0), (8, 1, 64, (300, 1), 10, 50)])
def test_values_that_a_row_does_not_see(mh, dt, nh, nkv, hd, seqs, bad, window):
    """A token with inf in v (NaN in a 4-bit block) and in k: rows before it and rows whose window is past it
    are as without it; a row that sees it is not finite."""
    say(f"kv attention masked non-finite dt={dt} heads={nh}/{nkv}x{hd} {seqs} bad={bad} window={window}")
    rng = np.random.default_rng(9)
    b = Batch([seqs], 32, rng)
    pg = Pages(dt, nkv, hd, 32, b.n_pages, rng)
    pg.fill(b.pages[0], seqs[0], rng)
    clean = Pages(dt, nkv, hd, 32, b.n_pages, rng)
    clean.arr = [a.copy() for a in pg.arr]
    x = rng.standard_normal((nkv, hd)).astype(F32)
    x[:, 5], x[:, 40] = np.inf, np.nan
    for w in (0, 1):
        pg.put(b.pages[0], bad, w, x)
    pg.upload()
    q = rng.standard_normal((b.n_rows, nh * hd)).astype(F32)
    got = run_attention(pg, b, nh, q, 0.125, window)
    sees = {row: (bad <= pos and (not window or bad > pos - window)) for row, _, pos in b.rows()}
    compare(clean, b, nh, q, 0.125, window, None, got, rows={r for r, s in sees.items() if not s})
    for r, s in sees.items():
        if s:
            assert np.isnan(got[r]).any()
    # in v alone only its own dims (its 4-bit block's) are touched
    pg.arr = [a.copy() for a in clean.arr]
    x[:] = 1.0
    x[:, 5] = np.inf
    pg.put(b.pages[0], bad, 1, x)
    pg.upload()
    got = run_attention(pg, b, nh, q, 0.125, window)
    for r, s in sees.items():
        g = got[r].reshape(nh, hd)
        want = np.zeros(hd, bool)
        want[5 if dt == KV_F16 else slice(0, 32)] = s
        assert (np.isfinite(g) == ~want).all(), r
    compare(clean, b, nh, q, 0.125, window, None, got, rows={r for r, s in sees.items() if not s})
    pg.free(), clean.free(), b.free()


@pytest.mark.parametrize("dt", [KV_F16, KV_MXFP4])
@pytest.mark.parametrize("rows,sink", [(1, 1), (1, 0), (3, 1), (24, 1)])
def test_nan_in_a_run_of_tokens(mh, dt, rows, sink):
    """Keys of NaN through whole work units of a long sequence, a NaN query, or every key NaN: the rows that
    see one are NaN in that head, the other heads and sequences as without it."""
    say(f"kv attention runs of NaN dt={dt} rows={rows} sink={sink}")
    rng, nh, nkv, hd, n = np.random.default_rng(31), 16, 2, 64, 6000
    b = Batch([(n, rows), (50, 1)], 64, rng)
    clean = Pages(dt, nkv, hd, 64, b.n_pages, rng)
    for s, (m, _) in enumerate(b.seqs):
        clean.fill(b.pages[s], m, rng)
    q = rng.standard_normal((b.n_rows, nh * hd)).astype(F32)
    sk = rng.standard_normal(nh).astype(F32) if sink else None
    for run, query in (((10, 60), None), ((0, 94), None), ((90, 91), None), (None, 5)):
        pg = Pages(dt, nkv, hd, 64, b.n_pages, rng)
        pg.arr = [a.copy() for a in clean.arr]
        if run:
            pg.arr[2 if dt == KV_MXFP4 else 0][b.pages[0][run[0]:run[1]], 1] = 255 if dt == KV_MXFP4 else 0x7E00
        x = q.copy()
        if query is not None:
            x[0].reshape(nh, hd)[query, 7] = np.nan
        pg.upload()
        got = run_attention(pg, b, nh, x, 0.125, 0, sk)
        nan = np.zeros((b.n_rows, nh), bool)
        if run:
            nan[:rows, nh // 2:] = True
        else:
            nan[0, query] = True
        assert (np.isnan(got.reshape(b.n_rows, nh, hd)) == nan[:, :, None]).all(), (run, query)
        clean.upload()
        plain = run_attention(clean, b, nh, q, 0.125, 0, sk)
        assert (got.reshape(b.n_rows, nh, hd)[~nan] == plain.reshape(b.n_rows, nh, hd)[~nan]).all()
        pg.free()
    clean.free(), b.free()


@pytest.mark.parametrize("rows,group,n", [(1, 8, 700), (2, 2, 300), (5, 8, 1100)])
def test_many_sequences(mh, rows, group, n):
    """More sequences than one look over them takes; lengths from nothing up, empty and padding rows among them."""
    say(f"kv attention {n} sequences of {rows} rows")
    rng = np.random.default_rng(n)
    nkv, hd, page = 1, 32, 16
    seqs = [(int(rng.integers(0, 90)), int(rng.integers(0, rows + 1)) if rows > 1 else 1) for _ in range(n)]
    seqs[5], seqs[n - 1] = (0, rows), (400, rows)
    b = Batch(seqs, page, rng, one=rows == 1)
    pg = Pages(KV_F16, nkv, hd, page, b.n_pages, rng)
    for s, (m, _) in enumerate(seqs):
        pg.fill(b.pages[s], m, rng)
    pg.upload()
    q = rng.standard_normal((b.n_rows, group * hd)).astype(F32)
    got = run_attention(pg, b, group * nkv, q, 0.2)
    compare(pg, b, group * nkv, q, 0.2, 0, None, got)
    pg.free(), b.free()


def test_memory_of_the_program(mh):
    """Arrays that the program allocated itself (not mh_alloc), inside a captured call too; host memory is refused."""
    import ctypes as C
    from hip_graph import hip_call
    rng, nh, nkv, hd, n = np.random.default_rng(4), 8, 1, 64, 300
    say("kv attention on the program's own memory")
    b = Batch([(n, 2)], 64, rng)
    pg = Pages(KV_MXFP4, nkv, hd, 64, b.n_pages, rng)
    pg.fill(b.pages[0], n, rng)
    pg.upload()
    q = rng.standard_normal((2, nh * hd)).astype(F32)
    ptr = [C.c_void_p() for _ in range(3)]
    need = kv.attention_ws(pg.cache, b.batch, nh)
    for p, size in zip(ptr, (q.nbytes, q.nbytes, need)):
        hip_call("hipMalloc", C.byref(p), C.c_size_t(size))
    hip_call("hipMemcpy", ptr[0], C.c_void_p(q.ctypes.data), C.c_size_t(q.nbytes), 1)
    out = np.zeros_like(q)

    def call():
        kv.attention_dev(pg.cache, b.batch, nh, ptr[0].value, ptr[1].value, ptr[2].value, need, 0.125)
    call()
    sync()
    hip_call("hipMemcpy", C.c_void_p(out.ctypes.data), ptr[1], C.c_size_t(q.nbytes), 2)
    compare(pg, b, nh, q, 0.125, 0, None, out)
    st = Stream()
    g = Graph(st, call)
    for _ in range(3):
        hip_call("hipMemset", ptr[1], 0, C.c_size_t(q.nbytes))
        hip_call("hipDeviceSynchronize")
        g.launch(st)
        st.sync()
        again = np.zeros_like(q)
        hip_call("hipMemcpy", C.c_void_p(again.ctypes.data), ptr[1], C.c_size_t(q.nbytes), 2)
        assert (again == out).all()
    for bad in (dict(q=q.ctypes.data & ~15), dict(out=q.ctypes.data & ~15), dict(ws=q.ctypes.data & ~15)):
        a = dict(q=ptr[0].value, out=ptr[1].value, ws=ptr[2].value)
        a.update(bad)
        with pytest.raises(MidgeHipError):
            kv.attention_dev(pg.cache, b.batch, nh, a["q"], a["out"], a["ws"], need, 0.125)
    # a result past the end of its allocation
    with pytest.raises(MidgeHipError):
        kv.attention_dev(pg.cache, b.batch, nh, ptr[0].value, ptr[1].value + 4096, ptr[2].value, need, 0.125)
    g.free(), st.free()
    for p in ptr:
        hip_call("hipFree", p)
    pg.free(), b.free()


@pytest.mark.parametrize("dt", [KV_F16, KV_MXFP4])
def test_overlaps_are_refused(mh, dt):
    """Outputs or workspace in the cache's memory, k and v in one place: refused, nothing written."""
    say(f"kv overlaps dt={dt}")
    rng, nh, nkv, hd, n = np.random.default_rng(5), 4, 2, 64, 600
    b = Batch([(n, 2)], 16, rng)
    pg = Pages(dt, nkv, hd, 16, b.n_pages, rng)
    dev = Dev()
    q, k, out = dev(np.zeros((2, nh * hd), F32)), dev(np.zeros((2, nkv * hd), F32)), dev(np.zeros((2, nh * hd), F32))
    need = kv.attention_ws(pg.cache, b.batch, nh)
    ws = dev(np.zeros(need, np.uint8))

    def refused(f, *a):
        with pytest.raises(MidgeHipError, match="overlap"):
            f(*a)

    def append(cache=pg.cache, q=q, k=k, v=k, out=out):
        kv.append_dev(cache, b.batch, KVRows(nh, 1, 1e-5, q, k, v, nh * hd, nkv * hd, nkv * hd, out))
    for inside in pg.bufs:
        refused(kv.attention_dev, pg.cache, b.batch, nh, q, inside, ws, need, 0.125)
        refused(kv.read_dev, pg.cache, b.batch, inside, None)
        refused(kv.read_dev, pg.cache, b.batch, None, inside)
        for name in ("q", "k", "v", "out"):
            refused(lambda: append(**{name: inside}))
    small = Batch([(1, 1)], 16, rng, n_pages=1)
    big = dev(np.zeros(kv.attention_ws(pg.cache, small.batch, nh) + pg.arr[0].nbytes, np.uint8))
    one = kv.KVCache(dt, nkv, hd, 16, 1, big, *pg.bufs[1:])
    refused(kv.attention_dev, one, small.batch, nh, q, out, big, kv.attention_ws(one, small.batch, nh), 0.125)
    refused(lambda: append(cache=kv.KVCache(dt, nkv, hd, 16, b.n_pages, pg.bufs[0], pg.bufs[0], *pg.bufs[2:])))
    if dt == KV_MXFP4:
        refused(lambda: append(cache=kv.KVCache(dt, nkv, hd, 16, b.n_pages, *pg.bufs[:2], pg.bufs[2], pg.bufs[2])))
        refused(lambda: append(cache=kv.KVCache(dt, nkv, hd, 16, b.n_pages, *pg.bufs[:2], pg.bufs[0], pg.bufs[3])))
    assert all((a == g).all() for a, g in zip(pg.arr, pg.download()))
    append()
    sync()
    dev.free(pg, b, small)


def test_bad_batches_are_reported(mh):
    """Page numbers, rows and lengths out of bounds: that sequence only, no access out of bounds, one error."""
    rng, nh, nkv, hd = np.random.default_rng(2), 8, 2, 64
    for what in ("page", "negative page", "len", "rows"):
        for rows in (1, 40):
            say(f"kv attention bad {what} rows={rows}")
            b = Batch([(100, rows), (90, rows), (130, rows)], 32, rng)
            pg = Pages(KV_MXFP4, nkv, hd, 32, b.n_pages, rng)
            for s, (n, _) in enumerate(b.seqs):
                pg.fill(b.pages[s], n, rng)
            pg.upload()
            good = [a.copy() for a in (b.row0, b.len, b.pages)]
            if what == "page":
                b.pages[1, 1] = b.n_pages
            elif what == "negative page":
                b.pages[1, 0] = -2
            elif what == "len":
                b.len[1] = b.max_pages * 32 + 1
            else:
                b.row0[-1] += 1         # past the arrays: the last sequence
            b.upload()
            q = rng.standard_normal((b.n_rows, nh * hd)).astype(F32)
            dev = Dev()
            with pytest.raises(MidgeHipError, match="out of bounds"):
                run_attention(pg, b, nh, q, 0.125, dev=dev)
            got = dev.bufs[0].download(F32, (b.n_rows, nh * hd))
            b.row0, b.len, b.pages = good
            hurt = 2 if what == "rows" else 1
            mine = set(range(b.row0[hurt], b.row0[hurt + 1]))
            compare(pg, b, nh, q, 0.125, 0, None, got, rows=set(range(b.n_rows)) - mine)
            for r in mine:
                if "page" in what:
                    assert np.isnan(got[r]).all()
                else:
                    assert (got[r] == 7.5).all()
            b.upload()
            dev.free()
            run_attention(pg, b, nh, q, 0.125)      # and nothing is left over
            pg.free(), b.free()
    say("kv append and read with a bad page")
    b = Batch([(20, 2), (40, 2)], 16, rng)
    pg = Pages(KV_F16, 2, hd, 16, b.n_pages, rng)
    b.pages[1, 2] = b.n_pages + 5
    b.upload()
    dev = Dev()
    x = rng.standard_normal((4, 2 * hd)).astype(F32)
    d, qo, ko = dev(x), dev(np.zeros_like(x)), dev(np.full_like(x, 7.5))
    kv.append_dev(pg.cache, b.batch, KVRows(2, 1, EPS, d, d, d, 2 * hd, 2 * hd, 2 * hd, qo))
    with pytest.raises(MidgeHipError, match="out of bounds"):
        sync()
    for row in (0, 1):
        for w in (0, 1):
            pg.put(b.pages[0], 18 + row, w, x[row].reshape(2, hd))
    assert all((a == g).all() for a, g in zip(pg.arr, pg.download()))
    assert (qo.download(F32, x.shape) == x).all()
    kv.read_dev(pg.cache, b.batch, ko, None)
    with pytest.raises(MidgeHipError, match="out of bounds"):
        sync()
    g = ko.download(F32, x.shape)
    assert (g[2:] == 7.5).all() and (g[:2] == f16(x[:2])).all()
    dev.free(pg, b)


@pytest.mark.parametrize("rows", [1, 5, 30])
def test_shared_pages(mh, rows):
    """Sequences on the same first pages (a common prompt), and one that has a page twice."""
    say(f"kv attention on shared pages rows={rows}")
    rng, nh, nkv, hd, page = np.random.default_rng(12), 16, 2, 128, 32
    b = Batch([(300, rows), (333, rows), (290, rows), (130, rows)], page, rng)
    b.pages[1, :8] = b.pages[2, :8] = b.pages[0, :8]
    b.pages[3, 2] = b.pages[3, 0]
    b.upload()
    for dt in (KV_F16, KV_MXFP4):
        pg = Pages(dt, nkv, hd, page, b.n_pages, rng)
        for s, (n, _) in enumerate(b.seqs):
            pg.fill(b.pages[s], n, rng)
        pg.upload()
        q = rng.standard_normal((b.n_rows, nh * hd)).astype(F32)
        got = run_attention(pg, b, nh, q, 0.09)
        compare(pg, b, nh, q, 0.09, 0, None, got)
        pg.free()
    b.free()


@pytest.mark.parametrize("rows", [1, 70])
def test_many_heads(mh, rows):
    """1024 k/v heads, and one head of its own for each of 300 query heads."""
    rng = np.random.default_rng(13)
    for nh, nkv, hd in ((1024, 1024, 32), (300, 300, 64)):
        say(f"kv append, attention and read of {nkv} k/v heads rows={rows}")
        b = Batch([(rows + 20, rows)], 16, rng)
        pg = Pages(KV_MXFP4, nkv, hd, 16, b.n_pages, rng)
        pg.fill(b.pages[0], rows + 20, rng)
        pg.upload()
        dev = Dev()
        x = [rng.standard_normal((rows, w * hd)).astype(F32) for w in (nh, nkv, nkv)]
        qo, ko, vo = dev(np.zeros((rows, nh * hd), F32)), dev(np.zeros((rows, nkv * hd), F32)), dev(np.zeros((rows, nkv * hd), F32))
        kv.append_dev(pg.cache, b.batch, KVRows(nh, 1, EPS, *[dev(a) for a in x], nh * hd, nkv * hd, nkv * hd, qo))
        kv.read_dev(pg.cache, b.batch, ko, vo)
        sync()
        assert (qo.download(F32, x[0].shape) == x[0]).all()
        for i in range(rows):
            for w in (0, 1):
                pg.put(b.pages[0], 20 + i, w, x[1 + w][i].reshape(nkv, hd))
        assert all((a == g).all() for a, g in zip(pg.arr, pg.download()))
        for w, buf in ((0, ko), (1, vo)):
            assert (buf.download(F32, (rows, nkv, hd)) == np.moveaxis(pg.tokens(b.pages[0], rows + 20, w)[:, 20:], 0, 1)).all()
        got = run_attention(pg, b, nh, x[0], 0.15)
        compare(pg, b, nh, x[0], 0.15, 0, None, got)
        dev.free(pg, b)


@pytest.mark.parametrize("rows", [2, 40])
def test_sequences_that_share_rows(mh, rows):
    """Row ranges that go back and forth, each valid by itself and together more than the call has rows: reported,
    nothing written past the workspace or the output."""
    say(f"kv attention, append and read of sequences that share rows={rows}")
    rng, nh, nkv, hd, n = np.random.default_rng(6), 8, 1, 64, 400
    b = Batch([(70, rows)] + [(70, 0)] * (n - 1), 32, rng)
    b.row0[:] = np.arange(n + 1) % 2 * rows
    b.upload()
    pg = Pages(KV_F16, nkv, hd, 32, b.n_pages, rng)
    dev, room = Dev(), 1 << 20
    need = kv.attention_ws(pg.cache, b.batch, nh)
    q, k = dev(rng.standard_normal((rows, nh * hd)).astype(F32)), dev(rng.standard_normal((rows, hd)).astype(F32))
    out, qo, ko = (dev(np.full(m + room // 4, 7.5, F32)) for m in (rows * nh * hd, rows * nh * hd, rows * hd))
    ws = dev(np.full(need + room, 0x5A, np.uint8))
    kv.attention_dev(pg.cache, b.batch, nh, q, out, ws, need, 0.125)
    with pytest.raises(MidgeHipError, match="out of bounds"):
        sync()
    with contextlib.suppress(MidgeHipError):   # (these look at the sequences that they find for their rows)
        kv.append_dev(pg.cache, b.batch, KVRows(nh, 1, EPS, q, k, k, nh * hd, hd, hd, qo))
        kv.read_dev(pg.cache, b.batch, ko, None)
        sync()
    assert (ws.download(np.uint8, (need + room,))[need:] == 0x5A).all()
    for buf, m in ((out, rows * nh * hd), (qo, rows * nh * hd), (ko, rows * hd)):
        assert (buf.download(F32, (m + room // 4,))[m:] == 7.5).all()
    dev.free(pg, b)


@pytest.mark.parametrize("dt", [KV_F16, KV_MXFP4])
def test_pages_past_4_gib(mh, dt):
    """Pages whose bytes lie past 32-bit offsets (the cache's memory is never written otherwise)."""
    nkv, hd, page = 8, 64, 256
    per = nkv * page * hd * (2 if dt == KV_F16 else 1) // (1 if dt == KV_F16 else 2)
    n_pages = (5 << 30) // per
    say(f"kv pages past 4 GiB dt={dt} n_pages={n_pages}")
    cache = kv.KVCache.alloc(dt, nkv, hd, page, n_pages)
    rng, dev = np.random.default_rng(1), Dev()
    n = 600
    pages = np.array([[n_pages - 1, n_pages - 7, n_pages // 2]], np.int32)
    b = Batch([(n, n)], page, rng)
    b.pages[:] = pages
    b.upload()
    k, v = [rng.standard_normal((n, nkv * hd)).astype(F32) for _ in "kv"]
    q = rng.standard_normal((n, 2 * nkv * hd)).astype(F32)
    dq, dk, dv = dev(q), dev(k), dev(v)
    kv.append_dev(cache, b.batch, KVRows(2 * nkv, 1, EPS, dq, dk, dv, 2 * nkv * hd, nkv * hd, nkv * hd, dq))
    ko, vo = dev(np.zeros_like(k)), dev(np.zeros_like(v))
    kv.read_dev(cache, b.batch, ko, vo)
    small = Pages(dt, nkv, hd, page, 3, rng)
    b.pages[:] = [[2, 0, 1]]
    for t in range(n):
        for w, x in ((0, k), (1, v)):
            small.put(b.pages[0], t, w, x[t].reshape(nkv, hd))
    for w, o in ((0, ko), (1, vo)):
        want = small.tokens(b.pages[0], n, w).transpose(1, 0, 2).reshape(n, -1)
        assert (o.download(F32, k.shape) == want).all()
    ws_n = kv.attention_ws(cache, b.batch, 2 * nkv)
    ws, out = dev(np.zeros(ws_n, np.uint8)), dev(np.zeros_like(q))
    kv.attention_dev(cache, b.batch, 2 * nkv, dq, out, ws, ws_n, 0.125)
    sync()
    compare(small, b, 2 * nkv, q, 0.125, 0, None, out.download(F32, q.shape), rows={0, 5, 300, 599})
    dev.free(small, b, cache)


# ------------------------------------------------------ streams and graphs

@pytest.mark.parametrize("rows", [1, 40])
def test_captured_and_replayed(mh, rows):
    """Append, attention and read in a captured graph: replays with new lengths, pages and rows, between the
    program's own calls, equal the eager results; two graphs on two streams with a workspace each."""
    nh, nkv, hd, page = 16, 2, 64, 32
    rng = np.random.default_rng(rows)
    graphs = []
    for dt in (KV_F16, KV_MXFP4):
        say(f"kv capture dt={dt} rows={rows}")
        b = Batch([(900, rows), (40, rows)], page, rng, max_pages=40, n_pages=90)
        pg = Pages(dt, nkv, hd, page, 90, rng)
        for s, (n, _) in enumerate(b.seqs):
            pg.fill(b.pages[s], n, rng)
        pg.upload()
        dev = Dev()
        n = b.n_rows
        co, si = tables(1300, hd)
        bufs = dict(q=dev(np.zeros((n, nh * hd), F32)), k=dev(np.zeros((n, nkv * hd), F32)), v=dev(np.zeros((n, nkv * hd), F32)),
                    qo=dev(np.zeros((n, nh * hd), F32)), out=dev(np.zeros((n, nh * hd), F32)), ko=dev(np.zeros((n, nkv * hd), F32)))
        r = KVRows(nh, 1300, EPS, bufs["q"], bufs["k"], bufs["v"], nh * hd, nkv * hd, nkv * hd, bufs["qo"], rope_cos=dev(co), rope_sin=dev(si))
        wn = kv.attention_ws(pg.cache, b.batch, nh)
        ws = dev(np.zeros(wn, np.uint8))

        def step(pg=pg, b=b, r=r, bufs=bufs, ws=ws, wn=wn):
            kv.append_dev(pg.cache, b.batch, r)
            kv.attention_dev(pg.cache, b.batch, nh, bufs["qo"], bufs["out"], ws, wn, 0.125)
            kv.read_dev(pg.cache, b.batch, bufs["ko"], None)

        sync()
        st = Stream()
        graphs.append((Graph(st, step), st, step, pg, b, bufs, dev))
    for it in range(4):
        for g, st, step, pg, b, bufs, dev in graphs:
            # new rows at new positions
            b.seqs = [(900 + 37 * it, rows), (40 + 200 * it, rows)]
            b.len[:] = [x for x, _ in b.seqs]
            order = np.random.default_rng(it).permutation(90)
            for s, at in ((0, 0), (1, 40)):
                b.pages[s] = order[at:at + 40]
            b.upload()
            for s, (x, _) in enumerate(b.seqs):
                pg.fill(b.pages[s], x, rng)
            pg.upload()
            for k in "qkv":
                shape = (b.n_rows, (nh if k == "q" else nkv) * hd)
                bufs[k].upload(rng.standard_normal(shape).astype(F32))
        for g, st, *_ in graphs:        # both in flight
            g.launch(st)
        for g, st, *_ in graphs:
            st.sync()
        for g, st, step, pg, b, bufs, dev in graphs:
            names = dict(out=nh, ko=nkv, qo=nh)
            got = {k: bufs[k].download(F32, (b.n_rows, w * hd)) for k, w in names.items()}
            mem = pg.download()
            for k, w in names.items():
                bufs[k].upload(np.zeros((b.n_rows, w * hd), F32))
            step()
            sync()
            for k, w in names.items():
                assert (got[k] == bufs[k].download(F32, (b.n_rows, w * hd))).all(), (it, k)
            assert all((x == y).all() for x, y in zip(mem, pg.download()))
    for g, st, step, pg, b, bufs, dev in graphs:
        dev.free(pg, b, g, st)


@pytest.mark.parametrize("rows", [1, 40])
def test_same_bits_again(mh, rows):
    """Two calls give the same bits, also with another call of other sizes between them."""
    rng, nh, nkv, hd = np.random.default_rng(6), 64, 8, 64
    say(f"kv attention repeated rows={rows}")
    b = Batch([(3000, rows), (100, rows), (1500, rows)], 64, rng)
    pg = Pages(KV_MXFP4, nkv, hd, 64, b.n_pages, rng)
    for s, (n, _) in enumerate(b.seqs):
        pg.fill(b.pages[s], n, rng)
    pg.upload()
    q = rng.standard_normal((b.n_rows, nh * hd)).astype(F32)
    dev = Dev()
    n = kv.attention_ws(pg.cache, b.batch, nh)
    ws, dq, out = dev(np.zeros(n, np.uint8)), dev(q), dev(np.zeros_like(q))
    got = []
    for i in range(4):
        kv.attention_dev(pg.cache, b.batch, nh, dq, out, ws, n, 0.125)
        sync()
        got.append(out.download(F32, q.shape))
        kv.attention_dev(pg.cache, b.batch, nh, dq, out, ws, n, 0.1, 64)
    assert all((g == got[0]).all() for g in got)
    compare(pg, b, nh, q, 0.125, 0, None, got[0], rows={0, rows, 2 * rows})
    dev.free(pg, b)


# ------------------------------------------------------------------ together

@pytest.mark.parametrize("window", [0, 24])
def test_layer_with_a_paged_cache(mh, window):
    """The attention layer of a prompt and some decode steps on a paged f16 cache (norm, projections of the
    whole chunk, append, attention, output projection, residual) against mh_attention_dev token by token."""
    from attn_dev import attn_device_layer
    from midge_amd import _lib
    from midge_amd.kern import WT, matvec_dev, rmsnorm_dev
    from test_oracle_kernels import AttnHost
    import ctypes as C
    say(f"attention layer on a paged cache, window {window}")
    cfg = dict(hidden=512, nh=16, nkv=4, hd=64, ctx=96, window=window, qk_norm=1, sinks=1)
    host = AttnHost(**cfg, seed=3)
    D, bufs, kc, vc = attn_device_layer(host, cfg)
    H, nh, nkv, hd = 512, 16, 4, 64
    steps = [40, 1, 1, 7, 1]        # a prompt, tokens, a chunk, a token
    total = sum(steps)
    rng, dev = np.random.default_rng(0), Dev()
    x = rng.standard_normal((total, H)).astype(F32)
    want = x.copy()
    row = dev(x[0])
    for t in range(total):
        row.upload(x[t])
        _lib.call("mh_attention_dev", C.byref(D), row.ptr, t)
        want[t] = row.download(F32, (H,))
    pages = rng.permutation(8).astype(np.int32)[None]
    cache = kv.KVCache.alloc(KV_F16, nkv, hd, 16, 8)
    wt = lambda w: WT(w.dt, w.rows, w.cols, w.data, w.scales)      # noqa: E731
    done, scale = 0, float(D.attn_scale)
    for n in steps:
        d_row0, d_len, d_pages = dev(np.array([0, n], np.int32)), dev(np.array([done + n], np.int32)), dev(pages)
        b = kv.KVBatch(1, n, n, 8, d_row0, d_len, d_pages)
        dx, xb = dev(x[done:done + n]), dev(np.zeros((n, H), F32))
        q, k, v = [dev(np.zeros((n, w * hd), F32)) for w in (nh, nkv, nkv)]
        ao, y = dev(np.zeros((n, nh * hd), F32)), dev(np.zeros((n, H), F32))
        rmsnorm_dev(dx, D.attn_norm, xb, H, float(D.norm_eps), n)
        for w, o in ((D.wq, q), (D.wk, k), (D.wv, v)):
            matvec_dev(wt(w), xb, o, n)
        kv.append_dev(cache, b, KVRows(nh, cfg["ctx"], float(D.norm_eps), q, k, v, nh * hd, nkv * hd, nkv * hd, q, D.bq, D.bk, D.bv, D.qn, D.kn,
                                       D.rope_cos, D.rope_sin))
        wn = kv.attention_ws(cache, b, nh)
        kv.attention_dev(cache, b, nh, q, ao, dev(np.zeros(wn, np.uint8)), wn, scale, window, D.sink)
        matvec_dev(wt(D.wo), ao, y, n)
        sync()
        bo = np.ctypeslib.as_array(C.cast(host.L.bo, C.POINTER(C.c_float)), (H,))
        got = x[done:done + n] + (y.download(F32, (n, H)) + bo)
        # a k or v next to a rounding border of f16 may fall on its other side (2^-11): the bar of the layer's own tests
        err = np.linalg.norm(got - want[done:done + n]) / np.linalg.norm(want[done:done + n] - x[done:done + n])
        assert err <= 1e-3, (done, n, err)
        done += n
    dev.free(cache, *bufs)


# ------------------------------------------------------- pages behind a window

@pytest.mark.parametrize("dt", [KV_F16, KV_MXFP4])
@pytest.mark.parametrize("nh,nkv,hd,rows", [(64, 8, 64, 1), (16, 1, 128, 1), (16, 4, 64, 5), (16, 2, 64, 70), (8, 1, 128, 40), (8, 1, 256, 40)])
@pytest.mark.parametrize("page,window", [(16, 128), (32, 20), (16, 1)])
def test_pages_behind_a_window(mh, dt, nh, nkv, hd, rows, page, window):
    """Pages that lie before every row's window, given back and marked out of bounds, at lengths of all alignments:
    no error, the results as before; the page of the first token that a row sees still counts."""
    say(f"kv attention pages behind a window dt={dt} heads={nh}/{nkv}x{hd} rows={rows} page={page} window={window}")
    rng = np.random.default_rng(page + window + rows)
    seqs = [(n + rows - 1, rows) for n in (300, 191, 192, 193, 200, 145, 161, 176, 129, 128, 40, 1, 259)]
    b = Batch(seqs, page, rng)
    pg = Pages(dt, nkv, hd, page, b.n_pages, rng)       # page 0 too may hold anything where it is nobody's
    for s, (n, _) in enumerate(seqs):
        pg.fill(b.pages[s], n, rng)
    pg.upload()
    q = rng.standard_normal((b.n_rows, nh * hd)).astype(F32)
    good = b.pages.copy()
    first = [max(0, n - r + 1 - window) for n, r in seqs]       # the first token that a sequence's first row sees
    for s, lo in enumerate(first):
        b.pages[s, :lo // page] = np.where(np.arange(lo // page) % 2, b.n_pages + 3, -1)
    b.upload()
    assert (b.pages != good).sum() > 20
    behind = b.pages.copy()
    got = run_attention(pg, b, nh, q, 0.125, window)
    b.pages = good
    compare(pg, b, nh, q, 0.125, window, None, got)
    # the first page that is seen, of one sequence
    b.pages = behind.copy()
    b.pages[0, first[0] // page] = -1
    b.upload()
    dev = Dev()
    with pytest.raises(MidgeHipError, match="out of bounds"):
        run_attention(pg, b, nh, q, 0.125, window, dev=dev)
    got = dev.bufs[0].download(F32, (b.n_rows, nh * hd))
    assert np.isnan(got[0]).all()
    b.pages = good
    compare(pg, b, nh, q, 0.125, window, None, got, rows=set(range(rows, b.n_rows)))
    dev.free(pg, b)


# ------------------------------------------------------------- many parts

@pytest.mark.parametrize("dt,nh,nkv,hd,rows,n", [
    # few rows: a sequence in 32 to 157 parts, more than one trip of the join takes
    (KV_MXFP4, 8, 1, 64, 1, 20000), (KV_F16, 8, 1, 64, 1, 20000), (KV_F16, 8, 1, 128, 1, 6000), (KV_MXFP4, 8, 1, 128, 1, 12000),
    (KV_MXFP4, 16, 1, 64, 1, 20000), (KV_F16, 8, 1, 128, 5, 6000), (KV_MXFP4, 8, 1, 96, 3, 12000), (KV_F16, 6, 1, 256, 2, 4000),
    # a chunk behind a long context: 17 and more parts, and more than 64
    (KV_MXFP4, 8, 1, 64, 16, 5000), (KV_F16, 8, 1, 64, 16, 20000), (KV_MXFP4, 8, 1, 64, 24, 20000), (KV_F16, 8, 1, 128, 16, 5000),
    (KV_MXFP4, 8, 1, 128, 16, 10000), (KV_F16, 8, 1, 96, 13, 9000), (KV_F16, 8, 1, 256, 16, 5000), (KV_F16, 16, 2, 64, 24, 6000)])
def test_sequences_in_many_parts(mh, dt, nh, nkv, hd, rows, n):
    """A long sequence that many blocks share, its scores rising or falling along it so that the parts' maxima differ:
    every part counts in the result."""
    say(f"kv attention in many parts dt={dt} heads={nh}/{nkv}x{hd} rows={rows} tokens={n}")
    rng = np.random.default_rng(n + hd)
    page = 64
    b = Batch([(n, rows)], page, rng)
    u = rng.standard_normal((nkv, 1, hd))
    u /= np.sqrt((u * u).mean(-1, keepdims=True))
    for name, rise in (("rising", 3.0), ("falling", -3.0), ("rising steeply", 25.0)):
        say(f"  scores {name}")
        pg = Pages(dt, nkv, hd, page, b.n_pages, rng)
        for t0 in range(0, n, page):
            m = min(page, n - t0)
            # q . k / sqrt(hd) gains `rise` along the sequence
            up = rise / np.sqrt(hd) * (t0 + np.arange(m))[None, :, None] / n
            for w, x in ((0, rng.standard_normal((nkv, m, hd)) * 0.3 + u * up), (1, rng.standard_normal((nkv, m, hd)))):
                at = (b.pages[0][t0 // page], slice(None), slice(0, m))
                if dt == KV_F16:
                    pg.arr[w][at] = f16(x.astype(F32)).view(np.uint16)
                else:
                    pg.arr[w][at], pg.arr[w + 2][at] = encode(x.astype(F32))
        pg.upload()
        q = (rng.standard_normal((rows, nkv, nh // nkv, hd)) * 0.3 + u[None]).reshape(rows, nh * hd).astype(F32)
        sk = rng.standard_normal(nh).astype(F32)
        got = run_attention(pg, b, nh, q, float(F32(hd ** -0.5)), 0, sk)
        worst = compare(pg, b, nh, q, float(F32(hd ** -0.5)), 0, sk, got)
        say(f"  worst error {worst:.3f} of the tolerance")
        pg.free()
    b.free()


@pytest.mark.parametrize("dt", [KV_F16, KV_MXFP4])
def test_weights_and_batches_under_the_cache_are_refused(mh, dt):
    """A bias, norm weight or rotation table, or the batch's own arrays, in memory that the append writes: refused,
    nothing written; the same call on memory of their own runs."""
    say(f"kv weights and batch arrays under what a call writes dt={dt}")
    rng, nh, nkv, hd, n = np.random.default_rng(15), 4, 2, 64, 600
    b = Batch([(n, 2)], 16, rng)
    pg = Pages(dt, nkv, hd, 16, b.n_pages, rng)
    dev = Dev()
    q, k, out = dev(np.zeros((2, nh * hd), F32)), dev(np.zeros((2, nkv * hd), F32)), dev(np.zeros((2, nh * hd), F32))
    co, si = (dev(t) for t in tables(n, hd))

    def append(batch=b.batch, **kw):
        kv.append_dev(pg.cache, batch, KVRows(nh, n, EPS, q, k, k, nh * hd, nkv * hd, nkv * hd, out, **{**dict(rope_cos=co, rope_sin=si), **kw}))

    def refused(**kw):
        with pytest.raises(MidgeHipError, match="overlap"):
            append(**kw)
    for inside in pg.bufs:
        if inside.nbytes >= n * hd * 2:         # (the tables are the longest)
            for name in ("rope_cos", "rope_sin"):
                refused(**{name: inside})
        for name in ("bq", "bk", "bv", "qn", "kn"):
            refused(**{name: inside})
        refused(batch=kv.KVBatch(1, 2, 2, b.max_pages, inside, *b.bufs[1:]))
        refused(batch=kv.KVBatch(1, 2, 2, b.max_pages, b.bufs[0], inside, b.bufs[2]))
        refused(batch=kv.KVBatch(1, 2, 2, b.max_pages, *b.bufs[:2], inside))
    assert all((a == g).all() for a, g in zip(pg.arr, pg.download()))
    append(bq=dev(np.ones(nh * hd, F32)))
    sync()
    dev.free(pg, b)


# ------------------------------------------------- calls that have few users

@pytest.mark.parametrize("dt", [KV_F16, KV_MXFP4])
@pytest.mark.parametrize("group,rows", [(300, 1), (300, 3), (129, 2), (7, 21)])
def test_wide_groups_and_rows_in_front(mh, dt, group, rows):
    """More query heads on a k/v head than a tile has columns; rows of no sequence before the first one's; sinks of
    every size, infinite ones among them."""
    say(f"kv attention group={group} rows={rows} dt={dt}")
    rng, nkv, hd, page = np.random.default_rng(group + rows), 2, 64, 32
    b = Batch([(200, rows), (1, rows), (70, 0), (333, rows)], page, rng, extra_rows=5)
    b.row0 += 3
    b.upload()
    pg = Pages(dt, nkv, hd, page, b.n_pages, rng)
    for s, (n, _) in enumerate(b.seqs):
        pg.fill(b.pages[s], n, rng)
    pg.upload()
    nh = group * nkv
    q = rng.standard_normal((b.n_rows, nh * hd)).astype(F32)
    sk = (rng.standard_normal(nh) * 3).astype(F32)
    sk[:4] = [-1e30, -np.inf, 60.0, -60.0]
    got = run_attention(pg, b, nh, q, 0.125, 0, sk)
    compare(pg, b, nh, q, 0.125, 0, sk, got)
    sk[:2] = [np.inf, 1e30]
    got = run_attention(pg, b, nh, q, 0.125, 0, sk)
    assert all((got[row].reshape(nh, hd)[:2] == 0).all() for row, _, _ in b.rows())
    pg.free(), b.free()


@pytest.mark.parametrize("dt", [KV_F16, KV_MXFP4])
@pytest.mark.parametrize("rows", [1, 3])
def test_append_to_many_sequences(mh, dt, rows):
    """700 sequences, some without rows: each row finds its own place."""
    say(f"kv append to 700 sequences of at most {rows} rows dt={dt}")
    rng, nh, nkv, hd, page = np.random.default_rng(rows), 4, 2, 64, 16
    seqs = [(int(rng.integers(1, 60)), 1 if rows == 1 else int(rng.integers(0, rows + 1))) for _ in range(700)]
    b = Batch(seqs, page, rng, extra_rows=0 if rows == 1 else 4, one=rows == 1)
    if rows > 1:
        b.row0 += 2
        b.upload()
    pg, dev = Pages(dt, nkv, hd, page, b.n_pages, rng), Dev()
    n = b.n_rows
    x = [rng.standard_normal((n, w * hd)).astype(F32) for w in (nh, nkv, nkv)]
    qo, ko, vo = [dev(np.full((n, w * hd), 7.5, F32)) for w in (nh, nkv, nkv)]
    kv.append_dev(pg.cache, b.batch, KVRows(nh, 1, EPS, *[dev(a) for a in x], nh * hd, nkv * hd, nkv * hd, qo))
    kv.read_dev(pg.cache, b.batch, ko, vo)
    sync()
    want = [np.full(a.shape, 7.5, F32) for a in x]
    for row, s, pos in b.rows():
        if pos < 0:
            continue
        want[0][row] = x[0][row]
        for w in (1, 2):
            a = x[w][row].reshape(nkv, hd)
            pg.put(b.pages[s], pos, w - 1, a)
            want[w][row] = (f16(a) if dt == KV_F16 else decode(*encode(a))).ravel()
    assert all((a == g).all() for a, g in zip(pg.arr, pg.download()))
    for w, o in zip(want, (qo, ko, vo)):
        assert (o.download(F32, w.shape) == w).all()
    dev.free(pg, b)


@pytest.mark.parametrize("dt,nh,nkv,hd,rows,n,bad", [(KV_F16, 32, 4, 128, 512, 16000, 15600), (KV_MXFP4, 64, 8, 64, 1000, 5000, 4990)])
def test_one_infinite_value_does_not_hold_a_call_up(mh, dt, nh, nkv, hd, rows, n, bad):
    """An inf in a late token's v of a prompt chunk: the rows before it as without it, in a time that a server can
    bear (0.1 s, a hundred times a call's own and more)."""
    import time
    say(f"kv attention one infinite value behind {n} tokens dt={dt}")
    rng = np.random.default_rng(n)
    b = Batch([(n, rows)], 128, rng)
    pg = Pages(dt, nkv, hd, 128, b.n_pages, rng)
    pg.fill(b.pages[0], n, rng)
    q = rng.standard_normal((b.n_rows, nh * hd)).astype(F32)
    clean = Pages(dt, nkv, hd, 128, b.n_pages, rng)
    clean.arr = [a.copy() for a in pg.arr]
    x = np.ones((nkv, hd), F32)
    x[:, 3] = np.inf
    pg.put(b.pages[0], bad, 1, x)
    pg.upload()
    dev = Dev()
    need = kv.attention_ws(pg.cache, b.batch, nh)
    dq, out, ws = dev(q), dev(np.full_like(q, 7.5)), dev(np.zeros(need, np.uint8))
    times = []
    for _ in range(3):
        t = time.perf_counter()
        kv.attention_dev(pg.cache, b.batch, nh, dq, out, ws, need, 0.1)
        sync()
        times.append(time.perf_counter() - t)
    say(f"  {min(times) * 1e3:.2f} ms")
    got = out.download(F32, q.shape)
    first = bad - (n - rows)        # the first row that sees it
    compare(clean, b, nh, q, 0.1, 0, None, got, rows={0, first // 2, *range(first - 20, first)})
    assert np.isfinite(got[:first]).all() and not np.isfinite(got[first:]).all(-1).any()
    assert min(times) < 0.1
    dev.free(pg, clean, b)


@pytest.mark.parametrize("dt", [KV_F16, KV_MXFP4])
@pytest.mark.parametrize("rows", [1, 5, 40])
def test_small_weights_beside_a_large_one(mh, dt, rows):
    """A first token that takes nearly all of the probability and whose v is zero: what is left of the many others,
    2^k times less probable each, is off by 2^-34 of the largest each (half a step of an f16 subnormal under 2^9)
    beside what tolerance() counts of their own sum."""
    rng, nh, nkv, hd, n = np.random.default_rng(21), 8, 1, 64, 3000
    b = Batch([(n, rows)], 64, rng)
    for k in (8, 12, 16, 24, 32, 48):
        say(f"kv attention small weights dt={dt} rows={rows} 2^-{k}")
        pg = Pages(dt, nkv, hd, 64, b.n_pages, rng)
        one, first = np.ones((nkv, hd), F32), np.zeros((nkv, hd), F32)
        first[:, 0] = k
        for t in range(n):
            pg.put(b.pages[0], t, 0, first if t == 0 else 0 * one)
            pg.put(b.pages[0], t, 1, 0 * one if t == 0 else one)
        pg.upload()
        q = np.zeros((rows, nh, hd), F32)
        q[..., 0] = 1
        got = run_attention(pg, b, nh, q.reshape(rows, -1), float(np.log(2)))
        kk, v = [pg.tokens(b.pages[0], n, w) for w in (0, 1)]
        for row, _, pos in b.rows():
            want, mag = attention(q[row], kk[:, :pos + 1], v[:, :pos + 1], float(F32(np.log(2))), None)
            err = np.abs(got[row].reshape(nh, hd) - want)
            assert (err <= (pos + 1) * 2.0 ** -34 + tolerance(mag, want, pos + 1)).all(), (row, err.max(), want.max())
        pg.free()
    b.free()
