"""Trees of drafted tokens on paged k/v caches on the GPU: the append, the
attention and the move of the kept rows against their definitions in 64 bits
(kv_oracle, tree_oracle), over cache types, head layouts, page sizes, tree
shapes, windows and what other branches and stale slots may hold."""
import numpy as np
import pytest

from conftest import say
from midge_amd import MidgeHipError, sync
from midge_amd import kv
from hip_graph import Graph, Stream
from kv_oracle import KV_F16, KV_MXFP4, Batch, KVRows, Pages, attention, decode, prepared
from test_gpu_kv import EPS, F32, Dev, tables, tolerance
from tree_oracle import SHAPES, paths, seen, trees

pytestmark = pytest.mark.gpu


def tree_paths(b, parent):
    return [paths(parent[b.row0[s]:b.row0[s + 1]]) for s in range(len(b.seqs))]


def rows_of(b, parent):
    """(row, sequence, its place there, base, path) of every row of a sequence."""
    for s, ((n, r), pp) in enumerate(zip(b.seqs, tree_paths(b, parent))):
        for i in range(r):
            yield int(b.row0[s]) + i, s, i, n - r, pp[i]


# ------------------------------------------------------------------ append

@pytest.mark.parametrize("dt,nh,nkv,hd,page,seqs,norm,bias,rope,fused,extra", [
    (KV_MXFP4, 64, 8, 64, 64, [(1, 1)], 0, 1, 1, 0, 0),
    (KV_MXFP4, 64, 8, 64, 16, [(17, 17), (40, 3), (16, 1)], 0, 1, 1, 1, 2),
    (KV_F16, 32, 4, 128, 16, [(90, 64), (33, 1), (64, 64), (0, 0)], 1, 0, 1, 0, 0),
    (KV_MXFP4, 4, 4, 32, 32, [(70, 35), (0, 0), (5, 5)], 1, 1, 1, 1, 1),
    (KV_F16, 6, 2, 96, 128, [(200, 63)], 1, 1, 1, 1, 0),
    (KV_MXFP4, 6, 2, 96, 16, [(19, 7)], 0, 0, 1, 0, 0),
    (KV_MXFP4, 3, 1, 192, 64, [(65, 3), (64, 64)], 1, 0, 0, 1, 3),
    (KV_MXFP4, 8, 1, 256, 256, [(300, 47), (2, 2)], 1, 1, 1, 0, 0),
    (KV_F16, 8, 8, 64, 32, [(33, 33)], 0, 0, 0, 0, 0),
    (KV_F16, 4, 2, 64, 16, [(9, 1), (33, 1), (16, 1)], 0, 0, 1, 0, 0)])
@pytest.mark.parametrize("shape", SHAPES)
def test_append(mh, shape, dt, nh, nkv, hd, page, seqs, norm, bias, rope, fused, extra):
    say(f"tree append {shape} dt={dt} heads={nh}/{nkv}x{hd} page={page} seqs={seqs} norm={norm} bias={bias} rope={rope} fused={fused}")
    rng = np.random.default_rng(nh * hd + page)
    b, dev = Batch(seqs, page, rng, extra, one=all(r == 1 for _, r in seqs) and not extra), Dev()
    pg, parent = Pages(dt, nkv, hd, page, b.n_pages, rng), trees(seqs, shape, rng)
    n, (wq, wk) = b.n_rows, (nh * hd, nkv * hd)
    pad = 5 if fused else 0     # a row stride that keeps no row 16-byte aligned
    m = rng.standard_normal((n, wq + 2 * wk + pad)).astype(F32)
    q, k, v = m[:, :wq], m[:, wq:wq + wk], m[:, wq + wk:wq + 2 * wk]
    bq, bk, bv = [rng.standard_normal(w).astype(F32) if bias else None for w in (wq, wk, wk)]
    qn, kn = [(1 + 0.1 * rng.standard_normal(hd)).astype(F32) if norm else None for _ in "qk"]
    ctx = max(x for x, _ in seqs)
    co, si = tables(ctx, hd) if rope else (None, None)
    ptr = lambda a: dev(a).ptr if a is not None else 0     # noqa: E731
    qo = dev(np.full((n, wq), 7.5, F32))
    if fused:
        at, ld = ptr(m), [m.shape[1]] * 3
        src = [at, at + 4 * wq, at + 4 * (wq + wk)]
    else:
        src, ld = [ptr(a) for a in (q, k, v)], [wq, wk, wk]
    r = KVRows(nh, ctx, EPS, *src, *ld, qo, ptr(bq), ptr(bk), ptr(bv), ptr(qn), ptr(kn), ptr(co), ptr(si))
    kv.tree_append_dev(pg.cache, b.batch, dev(np.append(parent, [-1] * extra).astype(np.int32)), r)
    sync()
    want_q = np.full((n, wq), 7.5)
    for row, s, i, base, path in rows_of(b, parent):
        pos = base + len(path) - 1
        c, sn = (co[pos], si[pos]) if rope else (None, None)
        want_q[row] = prepared(q[row].reshape(nh, hd), bq, qn, EPS, c, sn).ravel()
        pg.put(b.pages[s], base + i, 0, prepared(k[row].reshape(nkv, hd), bk, kn, EPS, c, sn).astype(F32))
        pg.put(b.pages[s], base + i, 1, prepared(v[row].reshape(nkv, hd), bv, None, EPS, None, None).astype(F32))
    for a, g in zip(pg.arr, pg.download()):       # every other slot as it was, too
        assert (a == g).all(), (a != g).sum()
    gq = qo.download(F32, (n, wq)).astype(np.float64)
    assert (np.abs(gq - want_q) <= 2.0 ** -24 * np.abs(want_q) + 1e-38).all()       # one rounding of the 64-bit value
    dev.free(pg, b)


@pytest.mark.parametrize("dt", [KV_F16, KV_MXFP4])
def test_append_and_keep_of_many_trees(mh, dt):
    """400 trees of 0 to 64 rows, rows of no sequence in front and behind: each row finds its depth and its place."""
    say(f"tree append and keep of 400 trees dt={dt}")
    rng, nh, nkv, hd, page = np.random.default_rng(2), 2, 1, 64, 16
    seqs = [(int(r + rng.integers(0, 50)), int(r)) for r in rng.integers(0, 65, 400)]
    b, dev = Batch(seqs, page, rng, extra_rows=7), Dev()
    b.row0 += 4
    b.upload()
    pg, shapes = Pages(dt, nkv, hd, page, b.n_pages, rng), [SHAPES[i % 4] for i in range(400)]
    parent = np.concatenate([[9] * 4, *(trees([s], shape, rng) for s, shape in zip(seqs, shapes)), [-9] * 3]).astype(np.int32)   # (of no row: anything)
    x, (co, si) = [rng.standard_normal((b.n_rows, w * hd)).astype(F32) for w in (nh, nkv, nkv)], tables(128, hd)
    qo = dev(np.full((b.n_rows, nh * hd), 7.5, F32))
    kv.tree_append_dev(pg.cache, b.batch, dev(parent), KVRows(nh, 128, EPS, *[dev(a) for a in x], nh * hd, nkv * hd, nkv * hd, qo, rope_cos=dev(co),
                                                              rope_sin=dev(si)))
    sync()
    want = np.full((b.n_rows, nh * hd), 7.5)
    for row, s, i, base, path in rows_of(b, parent):
        pos = base + len(path) - 1
        want[row] = prepared(x[0][row].reshape(nh, hd), None, None, EPS, co[pos], si[pos]).ravel()
        pg.put(b.pages[s], base + i, 0, prepared(x[1][row].reshape(nkv, hd), None, None, EPS, co[pos], si[pos]).astype(F32))
        pg.put(b.pages[s], base + i, 1, x[2][row].reshape(nkv, hd))
    assert (np.abs(qo.download(F32, want.shape) - want) <= 2.0 ** -24 * np.abs(want)).all()
    assert all((a == g).all() for a, g in zip(pg.arr, pg.download()))
    kept, n_kept = np.full((400, b.max_rows), -1, np.int32), np.zeros(400, np.int32)
    after = [a.copy() for a in pg.arr]
    for s, (n, r) in enumerate(seqs):
        p = path_of(parent[b.row0[s]:b.row0[s + 1]], rng) if r else []
        n_kept[s], kept[s, :len(p)] = len(p), p
        for j, f in enumerate(p):
            for w, a in zip(after, pg.arr):
                w[b.pages[s, (n - r + j) // page], :, (n - r + j) % page] = a[b.pages[s, (n - r + f) // page], :, (n - r + f) % page]
    ln = dev(np.zeros(400, np.int32))
    kv.keep_dev([pg.cache], b.batch, dev(n_kept), dev(kept), ln)
    sync()
    assert all((a == g).all() for a, g in zip(after, pg.download()))
    assert (ln.download(np.int32, (400,)) == [n - r + k for (n, r), k in zip(seqs, n_kept)]).all()
    dev.free(pg, b)


def test_positions_past_the_tables(mh):
    """A row's depth counts against the rotation tables, not its place among the rows."""
    say("tree append, positions past the tables")
    rng, hd = np.random.default_rng(5), 64
    b, dev = Batch([(20, 6)], 16, rng), Dev()
    parent = np.array([-1, 0, 0, 1, 3, 0], np.int32)    # positions 14, 15, 15, 16, 17, 15
    pg = Pages(KV_F16, 2, hd, 16, b.n_pages, rng)
    co, si = tables(16, hd)
    q, k, v = [rng.standard_normal((6, w * hd)).astype(F32) for w in (4, 2, 2)]
    qo = dev(np.full_like(q, 7.5))
    kv.tree_append_dev(pg.cache, b.batch, dev(parent), KVRows(4, 16, EPS, dev(q), dev(k), dev(v), 4 * hd, 2 * hd, 2 * hd, qo, rope_cos=dev(co),
                                                             rope_sin=dev(si)))
    with pytest.raises(MidgeHipError, match="out of bounds"):
        sync()
    sync()      # said once
    want = np.full(q.shape, 7.5)
    for row, s, i, base, path in rows_of(b, parent):
        pos = base + len(path) - 1
        if pos < 16:
            want[row] = prepared(q[row].reshape(4, hd), None, None, EPS, co[pos], si[pos]).ravel()
            pg.put(b.pages[0], base + i, 0, prepared(k[row].reshape(2, hd), None, None, EPS, co[pos], si[pos]).astype(F32))
            pg.put(b.pages[0], base + i, 1, v[row].reshape(2, hd))
    assert (np.abs(qo.download(F32, q.shape) - want) <= 2.0 ** -24 * np.abs(want)).all()
    assert all((a == g).all() for a, g in zip(pg.arr, pg.download()))
    dev.free(pg, b)


# --------------------------------------------------------------- attention

def run(pg, b, parent, nh, q, scale, window=0, sink=None, dev=None):
    """(out with 7.5 where nothing was written)"""
    own = dev or Dev()
    out = own(np.full((b.n_rows, nh * pg.hd), 7.5, F32))
    n = kv.tree_attention_ws(pg.cache, b.batch, nh)
    ws = own(np.full(n + 4096, 0x5A, np.uint8))
    par = own(np.append(parent, [-1] * (b.n_rows - len(parent))).astype(np.int32))
    kv.tree_attention_dev(pg.cache, b.batch, par, nh, own(q), out, ws, n, scale, window, own(sink) if sink is not None else None)
    sync()
    assert (ws.download(np.uint8, (n + 4096,))[n:] == 0x5A).all()
    r = out.download(F32, (b.n_rows, nh * pg.hd))
    if dev is None:
        own.free()
    return r


def compare(pg, b, parent, nh, q, scale, window, sink, got, rows=None):
    cache, worst, written = {}, 0.0, np.zeros(b.n_rows, bool)
    for row, s, _, base, path in rows_of(b, parent):
        written[row] = True
        if rows is not None and row not in rows:
            continue
        if s not in cache:
            cache[s] = [pg.tokens(b.pages[s], b.seqs[s][0], w) for w in (0, 1)]
        at = seen(base, path, window)
        k, v = (x[:, at] for x in cache[s])
        want, mag = attention(q[row].reshape(nh, -1), k, v, scale, sink)
        err, tol = np.abs(got[row].reshape(nh, -1) - want).max(), tolerance(mag, np.abs(v).max(), len(at))
        assert err <= tol, (row, s, base, path, err, tol)
        worst = max(worst, err / tol)
    assert (got[~written] == 7.5).all()
    return worst


ATTEND = [
    # dt, nh, nkv, hd, page, seqs [(len, rows)], window, sink, extra rows
    (KV_MXFP4, 64, 8, 64, 64, [(1, 1)], 0, 1, 0),
    (KV_MXFP4, 64, 8, 64, 16, [(17, 5), (300, 3), (0, 0), (64, 1), (65, 6), (1000, 2), (6, 6)], 0, 1, 2),
    (KV_F16, 64, 8, 64, 64, [(1025, 4), (256, 4), (257, 3)], 128, 0, 0),
    (KV_MXFP4, 32, 8, 128, 32, [(777, 12), (31, 7), (4000, 12)], 0, 0, 0),
    (KV_F16, 32, 4, 128, 16, [(500, 2), (90, 3), (5, 5), (0, 0), (33, 1)], 0, 1, 1),
    (KV_MXFP4, 32, 4, 128, 64, [(500, 4), (4, 4)], 3, 1, 0),
    (KV_MXFP4, 4, 4, 32, 256, [(700, 48), (33, 33)], 0, 0, 0),
    (KV_F16, 16, 16, 64, 128, [(333, 40)], 5, 1, 0),
    (KV_MXFP4, 6, 2, 96, 16, [(257, 1), (100, 5)], 0, 1, 0),
    (KV_F16, 8, 1, 256, 16, [(129, 1), (64, 4)], 0, 1, 0),
    (KV_F16, 12, 4, 192, 64, [(200, 10)], 0, 0, 0),
    # more columns than the streaming kernel takes
    (KV_MXFP4, 64, 8, 64, 64, [(64, 64)], 0, 1, 0),
    (KV_MXFP4, 64, 8, 64, 16, [(200, 64), (33, 33), (1, 1), (0, 0), (500, 20), (16, 9)], 128, 1, 3),
    (KV_F16, 32, 8, 128, 128, [(300, 61), (90, 13)], 0, 0, 0),
    (KV_MXFP4, 32, 4, 128, 32, [(97, 57), (1200, 40)], 0, 1, 0),
    (KV_F16, 4, 4, 32, 16, [(290, 64)], 2, 0, 0),
    (KV_MXFP4, 6, 2, 96, 64, [(150, 64), (20, 20)], 0, 1, 0),
    (KV_F16, 24, 2, 96, 32, [(400, 33)], 7, 0, 0),
    (KV_MXFP4, 12, 4, 192, 64, [(140, 55)], 0, 0, 0),
    (KV_F16, 3, 1, 192, 64, [(120, 64)], 20, 1, 0),
    (KV_F16, 8, 1, 256, 16, [(129, 47)], 0, 1, 0),
    (KV_MXFP4, 8, 1, 256, 64, [(300, 33)], 1, 0, 0),
    (KV_MXFP4, 40, 1, 64, 64, [(222, 11)], 0, 0, 0),
    (KV_MXFP4, 16, 2, 64, 1024, [(2500, 17), (60, 60), (700, 60)], 0, 1, 2),
    (KV_F16, 16, 2, 64, 4096, [(1900, 50)], 900, 0, 0),
    (KV_MXFP4, 64, 8, 64, 2048, [(5000, 9), (3, 3), (2100, 8)], 0, 1, 0),
    (KV_F16, 300, 1, 64, 32, [(90, 3), (333, 2)], 0, 1, 0),
]
# every head width and type at the column counts between which the kernels change
ATTEND += [(dt, g * 2, 2, hd, 32, [(330, r), (70, 1), (r, r), (0, 0), (95, max(1, r - 1))], w, 1, 1)
           for dt in (KV_F16, KV_MXFP4) for hd in (32, 64, 96, 128, 192, 256) for g, r, w in ((1, 8, 0), (2, 5, 60), (4, 8, 0), (8, 6, 2), (8, 8, 0), (8, 16, 70), (13, 10, 0), (2, 64, 0))]


@pytest.mark.parametrize("dt,nh,nkv,hd,page,seqs,window,sink,extra", ATTEND)
def test_attention(mh, dt, nh, nkv, hd, page, seqs, window, sink, extra):
    rng = np.random.default_rng(nh * hd + page + len(seqs))
    b = Batch(seqs, page, rng, extra, one=all(r == 1 for _, r in seqs) and not extra)
    pg = Pages(dt, nkv, hd, page, b.n_pages, rng)       # stale slots hold anything, NaN and inf among it
    for s, (n, _) in enumerate(seqs):
        pg.fill(b.pages[s], n, rng)
    pg.upload()
    q = (rng.standard_normal((b.n_rows, nh * hd)) * 1.5).astype(F32)
    sk = rng.standard_normal(nh).astype(F32) if sink else None
    scale = float(F32(hd ** -0.5))
    for shape in SHAPES:
        say(f"tree attention {shape} dt={dt} heads={nh}/{nkv}x{hd} page={page} seqs={seqs} window={window} sink={sink}")
        parent = trees(seqs, shape, rng)
        worst = compare(pg, b, parent, nh, q, scale, window, sk, run(pg, b, parent, nh, q, scale, window, sk))
        say(f"  worst error {worst:.3f} of the tolerance")
    pg.free(), b.free()


@pytest.mark.parametrize("dt", [KV_F16, KV_MXFP4])
@pytest.mark.parametrize("rows", [1, 4, 24])
def test_hard_scores(mh, dt, rows):
    """Large scores (one token takes all), tiny and large q and v, a negative and a zero scale, a window of one."""
    rng, nh, nkv, hd, n = np.random.default_rng(11), 16, 2, 64, 700
    for qs, vs, scale, window in ((30.0, 1.0, 0.125, 0), (1e-6, 1.0, 0.125, 0), (1.0, 1e-3, 0.125, 0), (1.0, 3e3, -0.3, 0), (1.0, 1.0, 0.0, 0),
                                  (1e4, 1.0, 1e-4, 0), (1.0, 1.0, 0.125, 1)):
        say(f"tree attention hard dt={dt} rows={rows} q*{qs} v*{vs} scale={scale} window={window}")
        b = Batch([(n, rows)], 64, rng)
        parent = trees(b.seqs, "any", rng)
        pg = Pages(dt, nkv, hd, 64, b.n_pages, rng)
        for w, std in ((0, 1.0), (1, vs)):
            for t in range(n):
                pg.put(b.pages[0], t, w, (rng.standard_normal((nkv, hd)) * std).astype(F32))
        pg.upload()
        q = (rng.standard_normal((b.n_rows, nh * hd)) * qs).astype(F32)
        compare(pg, b, parent, nh, q, scale, window, None, run(pg, b, parent, nh, q, scale, window))
        pg.free(), b.free()


@pytest.mark.parametrize("dt", [KV_F16, KV_MXFP4])
@pytest.mark.parametrize("nh,nkv,hd,seqs,window", [
    (8, 1, 64, (1500, 5), 0), (8, 2, 64, (300, 9), 0), (8, 1, 128, (70, 6), 4), (64, 8, 64, (90, 64), 0), (4, 2, 128, (260, 60), 3), (8, 1, 256, (100, 30), 0),
    (16, 2, 64, (33, 33), 0)])
@pytest.mark.parametrize("bad", ["own", "other"])
def test_values_that_a_row_does_not_see(mh, dt, nh, nkv, hd, seqs, window, bad):
    """A tree's row with inf and NaN in k and v: rows of other branches are as without it; those on whose path (and in
    whose window) it lies are not finite. And a cached token that some rows' windows have passed."""
    rng = np.random.default_rng(9)
    b = Batch([seqs], 32, rng)
    n, rows = seqs
    base = n - rows
    clean = Pages(dt, nkv, hd, 32, b.n_pages, rng)
    clean.fill(b.pages[0], n, rng)
    parent = trees(b.seqs, "any", rng)
    pp = paths(parent)
    at = base + 2 if bad == "own" else max(0, base - (window or 1) + 2 if window else base - 1)
    say(f"tree attention non-finite dt={dt} heads={nh}/{nkv}x{hd} {seqs} token {at} window={window}")
    q = rng.standard_normal((b.n_rows, nh * hd)).astype(F32)
    sees = [at in seen(base, p, window) for p in pp]
    assert window or bad == "other" or not all(sees)
    for part in ("both", "v"):
        pg = Pages(dt, nkv, hd, 32, b.n_pages, rng)
        pg.arr = [a.copy() for a in clean.arr]
        x = rng.standard_normal((nkv, hd)).astype(F32)
        x[:, 5] = np.inf
        if part == "both":
            x[:, 40 % hd] = np.nan
            pg.put(b.pages[0], at, 0, x)
        pg.put(b.pages[0], at, 1, x)
        pg.upload()
        got = run(pg, b, parent, nh, q, 0.125, window)
        compare(clean, b, parent, nh, q, 0.125, window, None, got, rows={r for r, s in enumerate(sees) if not s})
        for r, s in enumerate(sees):
            g = got[r].reshape(nh, hd)
            if part == "both":
                assert np.isnan(g).any() == s
            else:       # only its own dims (its 4-bit block's) are touched
                want = np.zeros(hd, bool)
                want[5 if dt == KV_F16 else slice(0, 32)] = s
                assert (np.isfinite(g) == ~want).all(), r
        pg.free()
    clean.free(), b.free()


@pytest.mark.parametrize("rows", [3, 40])
def test_bad_batches(mh, rows):
    """A parent out of range counts as -1; a sequence shorter than its tree, or with a length past its pages, is left out; a page out of
    bounds makes NaN of the rows that see it. mh_sync says so each time, and nothing else is touched."""
    rng, nh, nkv, hd, page = np.random.default_rng(2), 16, 2, 64, 32
    seqs = [(300, rows), (rows + 5, rows), (90, rows - 1)]
    b = Batch(seqs, page, rng)
    good = (b.row0.copy(), b.len.copy(), b.pages.copy())
    clean = trees(seqs, "any", rng)
    pg = Pages(KV_F16, nkv, hd, page, b.n_pages, rng)
    for s, (n, _) in enumerate(seqs):
        pg.fill(b.pages[s], n, rng)
    pg.upload()
    q = rng.standard_normal((b.n_rows, nh * hd)).astype(F32)

    def bad_run(parent):
        dev = Dev()
        b.upload()
        with pytest.raises(MidgeHipError, match="out of bounds"):
            run(pg, b, parent, nh, q, 0.125, 0, None, dev)
        out = dev.bufs[0].download(F32, (b.n_rows, nh * hd))
        dev.free()
        return out
    for what, value in (("itself", 1), ("a later row", 2), ("before -1", -2), ("far", 1 << 30)):
        say(f"tree attention with a parent that is {what} rows={rows}")
        parent = clean.copy()
        parent[b.row0[1] + 1] = value
        compare(pg, b, parent, nh, q, 0.125, 0, None, bad_run(parent))       # (paths() takes it as -1)
    for what, value in (("shorter than its tree", rows - 1), ("negative", -1), ("past its pages", b.max_pages * page + 1)):
        say(f"tree attention with a length that is {what} rows={rows}")
        b.len[1] = value
        got = bad_run(clean)
        assert (got[b.row0[1]:b.row0[2]] == 7.5).all()
        b.len[1] = good[1][1]
        got[b.row0[1]:b.row0[2]] = 0        # (compare() looks at what it is told to, and at rows of no sequence)
        compare(pg, b, clean, nh, q, 0.125, 0, None, got, rows={*range(b.row0[1]), *range(b.row0[2], b.n_rows)})
    say(f"tree attention with a page out of bounds rows={rows}")
    b.pages[2, 1] = b.n_pages
    got = bad_run(clean)
    assert np.isnan(got[b.row0[2]:]).all()
    b.pages[:] = good[2]
    compare(pg, b, clean, nh, q, 0.125, 0, None, got, rows=set(range(b.row0[2])))
    pg.free(), b.free()


@pytest.mark.parametrize("dt", [KV_F16, KV_MXFP4])
@pytest.mark.parametrize("rows", [4, 20])
def test_chains_are_prompt_chunks(mh, dt, rows):
    """A chain's append gives the same bits as mh_kv_append_dev, its attention the same values."""
    say(f"tree of a chain dt={dt} rows={rows}")
    rng, nh, nkv, hd, page = np.random.default_rng(1), 16, 2, 64, 32
    seqs = [(300, rows), (rows, rows), (77, rows - 1)]
    b, dev = Batch(seqs, page, rng), Dev()
    n, parent, (co, si) = b.n_rows, dev(trees(seqs, "chain", rng)), tables(300, hd)
    x = [rng.standard_normal((n, w * hd)).astype(F32) for w in (nh, nkv, nkv)]
    got = []
    start = Pages(dt, nkv, hd, page, b.n_pages, rng, junk=False)
    for as_tree in (False, True):
        pg = Pages(dt, nkv, hd, page, b.n_pages, rng)
        pg.arr = [a.copy() for a in start.arr]
        pg.upload()
        qo, out = dev(np.zeros((n, nh * hd), F32)), dev(np.zeros((n, nh * hd), F32))
        r = KVRows(nh, 300, EPS, *[dev(a) for a in x], nh * hd, nkv * hd, nkv * hd, qo, rope_cos=dev(co), rope_sin=dev(si))
        need = kv.tree_attention_ws(pg.cache, b.batch, nh) if as_tree else kv.attention_ws(pg.cache, b.batch, nh)
        ws = dev(np.zeros(need, np.uint8))
        if as_tree:
            kv.tree_append_dev(pg.cache, b.batch, parent, r)
            kv.tree_attention_dev(pg.cache, b.batch, parent, nh, qo, out, ws, need, 0.125, 50)
        else:
            kv.append_dev(pg.cache, b.batch, r)
            kv.attention_dev(pg.cache, b.batch, nh, qo, out, ws, need, 0.125, 50)
        sync()
        got.append([*pg.download(), qo.download(F32, (n, nh * hd)), out.download(F32, (n, nh * hd))])
        pg.free()
    assert all((x == y).all() for x, y in zip(got[0][:-1], got[1][:-1]))
    v = decode(got[0][1], got[0][3]) if dt == KV_MXFP4 else got[0][1].view(np.float16).astype(np.float64)
    assert np.abs(got[0][-1] - got[1][-1]).max() <= 2 * tolerance(10.0, np.abs(v).max(), 300)
    dev.free(start, b)


# -------------------------------------------------------------------- keep

def path_of(parent, rng):
    """A path down a tree from its first row, as a verification keeps it."""
    out = [0]
    for i in range(1, len(parent)):
        if parent[i] == out[-1] and rng.random() < 0.8:
            out.append(i)
    return out


@pytest.mark.parametrize("dt,nkv,hd,page,layers", [
    (KV_F16, 8, 64, 16, 1), (KV_MXFP4, 8, 64, 16, 3), (KV_F16, 2, 256, 64, 2), (KV_MXFP4, 1, 32, 32, 70), (KV_MXFP4, 3, 96, 16, 2), (KV_F16, 4, 128, 128, 65),
    (KV_MXFP4, 2, 192, 16, 2), (KV_F16, 1, 96, 16, 1), (KV_MXFP4, 1, 256, 64, 1), (KV_F16, 300, 32, 16, 1)])
def test_keep(mh, dt, nkv, hd, page, layers):
    """Kept rows move, everything else stays; whole trees, nothing, first rows, any ascending rows, paths."""
    say(f"keep dt={dt} heads={nkv}x{hd} page={page} layers={layers}")
    rng = np.random.default_rng(hd + layers)
    seqs = [(100, 64), (70, 64), (40, 7), (16, 16), (0, 0), (33, 33), (90, 1), (64, 50), (200, 30)]
    b, dev = Batch(seqs, page, rng, extra_rows=2), Dev()
    parent = trees(seqs, "any", rng)
    kept, n_kept = np.full((len(seqs), b.max_rows), -7, np.int32), np.zeros(len(seqs), np.int32)
    for s, (_, r) in enumerate(seqs):
        rows = [list(range(r)), [], list(range(min(r, 3))), sorted(rng.choice(r, r // 2, replace=False)) if r else [], [], [32],
                [0], list(range(1, r)), path_of(parent[b.row0[s]:b.row0[s + 1]], rng)][s]
        n_kept[s], kept[s, :len(rows)] = len(rows), rows
    layer = [Pages(dt, nkv, hd, page, b.n_pages, rng) for _ in range(layers)]
    out = dev(np.full(len(seqs) + 2, 77, np.int32))
    kv.keep_dev([p.cache for p in layer], b.batch, dev(n_kept), dev(kept), out)
    sync()
    for p in layer:
        want = [a.copy() for a in p.arr]
        for s, (n, r) in enumerate(seqs):
            for j in range(n_kept[s]):
                to, frm = n - r + j, n - r + kept[s, j]
                for w, a in zip(want, p.arr):
                    w[b.pages[s, to // page], :, to % page] = a[b.pages[s, frm // page], :, frm % page]
        for w, g in zip(want, p.download()):
            assert (w == g).all()
    assert (out.download(np.int32, (len(seqs) + 2,)) == [*(n - r + k for (n, r), k in zip(seqs, n_kept)), 77, 77]).all()
    dev.free(b, *layer)


@pytest.mark.parametrize("what", ["n_kept", "negative", "row", "order", "twice", "page", "short"])
def test_keep_of_bad_sequences(mh, what):
    """A sequence with something out of bounds is left as it is, the others move, and mh_sync says so."""
    say(f"keep, bad {what}")
    rng, nkv, hd, page = np.random.default_rng(4), 2, 64, 16
    seqs = [(60, 20), (50, 20), (80, 10)]
    b, dev = Batch(seqs, page, rng), Dev()
    kept = np.array([[0, 3, 5, 9] + [-1] * 16] * 3, np.int32)
    n_kept = np.full(3, 4, np.int32)
    if what == "n_kept":
        n_kept[1] = 21
    elif what == "negative":
        n_kept[1] = -1
    elif what == "row":
        kept[1, 3] = 20
    elif what == "order":
        kept[1, :4] = [0, 5, 3, 9]
    elif what == "twice":
        kept[1, 2] = 3
    elif what == "page":
        b.pages[1, (30 + 9) // page] = b.n_pages
    else:
        b.len[1] = 19
    b.upload()
    pg = Pages(KV_MXFP4, nkv, hd, page, b.n_pages, rng)
    out = dev(np.full(3, 77, np.int32))
    kv.keep_dev([pg.cache], b.batch, dev(n_kept), dev(kept), out)
    with pytest.raises(MidgeHipError, match="out of bounds"):
        sync()
    want = [a.copy() for a in pg.arr]
    for s in (0, 2):
        n, r = seqs[s]
        for j, f in enumerate((0, 3, 5, 9)):
            for w, a in zip(want, pg.arr):
                w[b.pages[s, (n - r + j) // page], :, (n - r + j) % page] = a[b.pages[s, (n - r + f) // page], :, (n - r + f) % page]
    assert all((w == g).all() for w, g in zip(want, pg.download()))
    assert (out.download(np.int32, (3,)) == [44, 77, 74]).all()
    dev.free(pg, b)


# ------------------------------------------------------ streams and graphs

@pytest.mark.parametrize("rows", [5, 24])
def test_captured_and_replayed(mh, rows):
    """Append, attention and keep in a captured graph: replays with new lengths, pages, trees and kept rows, between the
    program's own calls, equal the eager results; two graphs on two streams with a workspace each."""
    nh, nkv, hd, page = 16, 2, 64, 32
    rng = np.random.default_rng(rows)
    graphs = []
    for dt in (KV_F16, KV_MXFP4):
        say(f"tree capture dt={dt} rows={rows}")
        b = Batch([(900, rows), (40, rows)], page, rng, max_pages=40, n_pages=90)
        pg = Pages(dt, nkv, hd, page, 90, rng)
        dev, n = Dev(), b.n_rows
        co, si = tables(1300, hd)
        bufs = dict(q=dev(np.zeros((n, nh * hd), F32)), k=dev(np.zeros((n, nkv * hd), F32)), v=dev(np.zeros((n, nkv * hd), F32)),
                    qo=dev(np.zeros((n, nh * hd), F32)), out=dev(np.zeros((n, nh * hd), F32)), parent=dev(np.full(n, -1, np.int32)),
                    n_kept=dev(np.zeros(2, np.int32)), kept=dev(np.zeros((2, b.max_rows), np.int32)), len=dev(np.zeros(2, np.int32)))
        r = KVRows(nh, 1300, EPS, bufs["q"], bufs["k"], bufs["v"], nh * hd, nkv * hd, nkv * hd, bufs["qo"], rope_cos=dev(co), rope_sin=dev(si))
        wn = kv.tree_attention_ws(pg.cache, b.batch, nh)
        ws = dev(np.zeros(wn, np.uint8))

        def step(pg=pg, b=b, r=r, bufs=bufs, ws=ws, wn=wn):
            kv.tree_append_dev(pg.cache, b.batch, bufs["parent"], r)
            kv.tree_attention_dev(pg.cache, b.batch, bufs["parent"], nh, bufs["qo"], bufs["out"], ws, wn, 0.125)
            kv.keep_dev([pg.cache], b.batch, bufs["n_kept"], bufs["kept"], bufs["len"])

        sync()
        st = Stream()
        graphs.append((Graph(st, step), st, step, pg, b, bufs, dev))
    for it in range(4):
        for g, st, step, pg, b, bufs, dev in graphs:
            b.seqs = [(900 + 37 * it, rows), (40 + 200 * it, rows - it)]
            b.len[:], b.row0[:] = [x for x, _ in b.seqs], [0, rows, 2 * rows - it]
            order = np.random.default_rng(it).permutation(90)
            for s, at in ((0, 0), (1, 40)):
                b.pages[s] = order[at:at + 40]
            b.upload()
            for s, (x, _) in enumerate(b.seqs):
                pg.fill(b.pages[s], x, rng)
            pg.upload()
            parent = np.append(trees(b.seqs, SHAPES[it], rng), [-1] * it).astype(np.int32)
            bufs["parent"].upload(parent)
            kept, n_kept = np.full((2, rows), -1, np.int32), np.zeros(2, np.int32)
            for s in (0, 1):
                p = path_of(parent[b.row0[s]:b.row0[s + 1]], rng)
                n_kept[s], kept[s, :len(p)] = len(p), p
            bufs["n_kept"].upload(n_kept), bufs["kept"].upload(kept)
            for k in "qkv":
                bufs[k].upload(rng.standard_normal((b.n_rows, (nh if k == "q" else nkv) * hd)).astype(F32))
        for g, st, *_ in graphs:        # both in flight
            g.launch(st)
        for g, st, *_ in graphs:
            st.sync()
        for g, st, step, pg, b, bufs, dev in graphs:
            names = dict(out=(b.n_rows, nh * hd), qo=(b.n_rows, nh * hd))
            got = {k: bufs[k].download(F32, w) for k, w in names.items()}
            ln, mem = bufs["len"].download(np.int32, (2,)), pg.download()
            for k, w in names.items():
                bufs[k].upload(np.zeros(w, F32))
            bufs["len"].upload(np.zeros(2, np.int32))
            pg.upload()
            step()
            sync()
            used = slice(0, int(b.row0[2]))
            for k, w in names.items():
                assert (got[k][used] == bufs[k].download(F32, w)[used]).all(), (it, k)
            assert (ln == bufs["len"].download(np.int32, (2,))).all() and all((x == y).all() for x, y in zip(mem, pg.download()))
    for g, st, step, pg, b, bufs, dev in graphs:
        dev.free(pg, b, g, st)


@pytest.mark.parametrize("rows", [5, 40])
def test_same_bits_again(mh, rows):
    """Two calls give the same bits, also with another call of other sizes between them."""
    rng, nh, nkv, hd = np.random.default_rng(6), 64, 8, 64
    say(f"tree attention repeated rows={rows}")
    b = Batch([(3000, rows), (100, rows), (1500, rows)], 64, rng)
    parent = trees(b.seqs, "any", rng)
    pg = Pages(KV_MXFP4, nkv, hd, 64, b.n_pages, rng)
    for s, (n, _) in enumerate(b.seqs):
        pg.fill(b.pages[s], n, rng)
    pg.upload()
    q, dev = rng.standard_normal((b.n_rows, nh * hd)).astype(F32), Dev()
    n = kv.tree_attention_ws(pg.cache, b.batch, nh)
    ws, dq, out, par, got = dev(np.zeros(n, np.uint8)), dev(q), dev(np.zeros_like(q)), dev(parent), []
    for _ in range(4):
        kv.tree_attention_dev(pg.cache, b.batch, par, nh, dq, out, ws, n, 0.125)
        sync()
        got.append(out.download(F32, q.shape))
        kv.tree_attention_dev(pg.cache, b.batch, par, nh, dq, out, ws, n, 0.1, 64)
    assert all((g == got[0]).all() for g in got)
    compare(pg, b, parent, nh, q, 0.125, 0, None, got[0], rows={0, rows, 2 * rows, 3 * rows - 1})
    dev.free(pg, b)


@pytest.mark.parametrize("dt", [KV_F16, KV_MXFP4])
@pytest.mark.parametrize("rows", [7, 30])
def test_trees_past_4_gib(mh, dt, rows):
    """Pages whose bytes lie past 32-bit offsets (the cache's memory is never written otherwise)."""
    nkv, hd, page = 8, 64, 256
    per = nkv * page * hd * (2 if dt == KV_F16 else 1) // (1 if dt == KV_F16 else 2)
    n_pages = (5 << 30) // per
    say(f"tree pages past 4 GiB dt={dt} rows={rows}")
    cache, rng, dev = kv.KVCache.alloc(dt, nkv, hd, page, n_pages), np.random.default_rng(1), Dev()
    b = Batch([(rows, rows)], page, rng)
    parent = trees(b.seqs, "any", rng)
    b.pages[:] = n_pages - 1
    b.upload()
    k, v = [rng.standard_normal((rows, nkv * hd)).astype(F32) for _ in "kv"]
    q = rng.standard_normal((rows, 2 * nkv * hd)).astype(F32)
    dq, par = dev(q), dev(parent)
    kv.tree_append_dev(cache, b.batch, par, KVRows(2 * nkv, 1, EPS, dq, dev(k), dev(v), 2 * nkv * hd, nkv * hd, nkv * hd, dq))
    need = kv.tree_attention_ws(cache, b.batch, 2 * nkv)
    out = dev(np.zeros_like(q))
    kv.tree_attention_dev(cache, b.batch, par, 2 * nkv, dq, out, dev(np.zeros(need, np.uint8)), need, 0.125)
    rowsk = path_of(parent, rng)
    ln, ko = dev(np.zeros(1, np.int32)), dev(np.zeros_like(k))
    kv.keep_dev([cache], b.batch, dev(np.array([len(rowsk)], np.int32)), dev(np.array(rowsk + [-1] * (rows - len(rowsk)), np.int32)), ln)
    kv.read_dev(cache, b.batch, ko, None)
    sync()
    small = Pages(dt, nkv, hd, page, 1, rng)
    b.pages[:] = 0
    for t in range(rows):
        for w, x in ((0, k), (1, v)):
            small.put(b.pages[0], t, w, x[t].reshape(nkv, hd))
    compare(small, b, parent, 2 * nkv, q, 0.125, 0, None, out.download(F32, q.shape))
    want = small.tokens(b.pages[0], rows, 0).transpose(1, 0, 2).reshape(rows, -1)
    want[:len(rowsk)] = want[rowsk]
    assert (ko.download(F32, k.shape) == want).all() and ln.download(np.int32, (1,))[0] == len(rowsk)
    dev.free(small, b, cache)


def test_empty_batches(mh):
    """No rows at all, and a batch in which no sequence has rows: nothing is written but lengths."""
    say("trees of no rows")
    rng, nh, nkv, hd, page = np.random.default_rng(2), 4, 2, 64, 16
    b, dev = Batch([(20, 0), (0, 0)], page, rng, extra_rows=3), Dev()
    pg = Pages(KV_F16, nkv, hd, page, b.n_pages, rng)
    out, x = dev(np.full((3, nh * hd), 7.5, F32)), dev(np.zeros((3, nh * hd), F32))
    for batch in (b.batch, kv.KVBatch(2, 0, 1, b.max_pages, *b.bufs)):
        need, par, ln = kv.tree_attention_ws(pg.cache, batch, nh), dev(np.full(3, -1, np.int32)), dev(np.zeros(2, np.int32))
        kv.tree_append_dev(pg.cache, batch, par, KVRows(nh, 1, EPS, x, x, x, nh * hd, nkv * hd, nkv * hd, out))
        kv.tree_attention_dev(pg.cache, batch, par, nh, x, out, dev(np.zeros(need, np.uint8)), need, 0.125)
        kv.keep_dev([pg.cache], batch, dev(np.zeros(2, np.int32)), dev(np.zeros((2, batch.c.max_rows), np.int32)), ln)
        sync()
        assert (out.download(F32, (3, nh * hd)) == 7.5).all() and (ln.download(np.int32, (2,)) == [20, 0]).all()
    assert all((a == g).all() for a, g in zip(pg.arr, pg.download()))
    dev.free(pg, b)
