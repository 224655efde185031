"""Attention of trees with 49 to 64 columns (rows x heads of a group) on up to
four sequences: the most that the kernel for few columns takes, and only for
trees. What each case asks of the dispatch is held by test_tree_few_host."""
import numpy as np
import pytest

from conftest import say
from kv_oracle import KV_F16, KV_MXFP4, Batch, Pages
from test_gpu_kv import F32
from test_gpu_kvtree import compare, run
from tree_oracle import SHAPES, paths, seen, trees

pytestmark = pytest.mark.gpu

# (heads of a group, rows): columns at both ends, of one row short of a wave's 16 columns, of a whole operand
COLUMNS = [(8, 7), (8, 8), (13, 4), (1, 64), (7, 7), (16, 4), (2, 31)]
# lengths behind which the rows lie: a tile and a part of one whole, one short, one more; none; parts of several blocks
SEQS = {1: [[64], [63], [1], [4100], [0]], 2: [[700, 5]], 4: [[130, 0, 2000, 64], [31, 1000, 1, 257]]}
CASES = [(dt, hd, g, r, n, base, w)
         for dt in (KV_F16, KV_MXFP4) for hd in (32, 64, 96, 128) for i, (g, r) in enumerate(COLUMNS)
         for n, base, w in ([(1, SEQS[1][i % 5], (0, 0, 3, 70)[i % 4]), (4, SEQS[4][i % 2], (0, 40)[i // 2 % 2])] + [(2, SEQS[2][0], 65)] * (i < 2))]
# the layout of most heads that the framework's models have, at lengths of many parts
CASES += [(dt, 64, 8, 8, 1, [n], w) for dt in (KV_F16, KV_MXFP4) for n, w in ((30000, 0), (9001, 0), (5000, 128))]


def batch_of(n, r, base, page, rng, extra=1):
    """`n` trees, the first of `r` rows, the others of fewer (one of none)."""
    rows = [r] + [max(0, r - k) if k < 3 else 0 for k in range(1, n)]
    return Batch([(b + m, m) for b, m in zip(base, rows)], page, rng, extra)


def heads_of(g, hd):
    return (2 if g * hd < 512 else 1) if hd != 64 else 8 if g == 8 else 3


@pytest.mark.parametrize("dt,hd,g,r,n,base,window", CASES)
def test_attention(mh, dt, hd, g, r, n, base, window):
    rng = np.random.default_rng(hd * g + r + n)
    nkv, page = heads_of(g, hd), (16, 64, 256)[(g + r) % 3]
    b = batch_of(n, r, base, page, rng)
    pg = Pages(dt, nkv, hd, page, b.n_pages, rng)       # stale slots hold anything, NaN and inf among it
    for s, (m, _) in enumerate(b.seqs):
        pg.fill(b.pages[s], m, rng)
    pg.upload()
    nh = nkv * g
    q = (rng.standard_normal((b.n_rows, nh * hd)) * 1.5).astype(F32)
    sk = rng.standard_normal(nh).astype(F32) if r % 2 else None
    for shape in SHAPES[:3] if max(base) < 9000 else SHAPES[:1]:
        say(f"trees of {g} x {r} columns {shape} dt={dt} hd={hd} heads={nkv} page={page} on {base} window={window}")
        parent = trees(b.seqs, shape, rng)
        compare(pg, b, parent, nh, q, float(F32(hd ** -0.5)), window, sk, run(pg, b, parent, nh, q, float(F32(hd ** -0.5)), window, sk))
    pg.free(), b.free()


ODD = [(dt, hd, g, r) for dt in (KV_F16, KV_MXFP4) for hd in (32, 64, 96, 128) for g, r in ((8, 8), (1, 64))]


@pytest.mark.parametrize("dt,hd,g,r", ODD)
def test_values_that_a_row_does_not_see(mh, dt, hd, g, r):
    """inf and NaN in a row of the tree, and in the last cached token behind a window of one: all 64 columns that do not
    see it are as without it, the others are not finite."""
    rng, nkv, n, page = np.random.default_rng(hd + r), 2, 333, 32
    b = Batch([(n, r)], page, rng)
    base, nh = n - r, nkv * g
    clean = Pages(dt, nkv, hd, page, b.n_pages, rng)
    clean.fill(b.pages[0], n, rng)
    parent = trees(b.seqs, "any", rng)
    pp = paths(parent)
    q = rng.standard_normal((b.n_rows, nh * hd)).astype(F32)
    for at, window in ((base + 2, 0), (base + r // 2, 0), (base - 1, 1)):
        sees = [at in seen(base, p, window) for p in pp]
        assert not all(sees)
        for which in (0, 1):
            say(f"trees of {g} x {r} columns, NaN and inf in {'kv'[which]} of token {at} dt={dt} hd={hd} window={window}")
            pg = Pages(dt, nkv, hd, page, b.n_pages, rng)
            pg.arr = [a.copy() for a in clean.arr]
            x = rng.standard_normal((nkv, hd)).astype(F32)
            x[:, 3], x[:, hd - 1] = np.inf, np.nan
            pg.put(b.pages[0], at, which, x)
            pg.upload()
            got = run(pg, b, parent, nh, q, 0.125, window)
            compare(clean, b, parent, nh, q, 0.125, window, None, got, rows={i for i, s in enumerate(sees) if not s})
            for i, s in enumerate(sees):
                assert np.isfinite(got[i]).all() != s, (at, i)
            pg.free()
    clean.free(), b.free()
