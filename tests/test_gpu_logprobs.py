"""mh_logprobs_dev against its definition in 64 bits."""
import numpy as np
import pytest

from conftest import say
from hip_graph import Graph, Stream
from midge_amd import DevBuf, MidgeHipError, sync
from midge_amd.moe import logprobs_dev, logprobs_ws

pytestmark = pytest.mark.gpu

F32 = np.float32


def oracle(x, ids, top):
    x64 = x.astype(np.float64)
    with np.errstate(all="ignore"):
        bad = np.isnan(x).any(-1) | (x == np.inf).any(-1)
        none = (x == -np.inf).all(-1)
        m = np.where(none | bad, 0, np.where(np.isnan(x64), -np.inf, x64).max(-1))[:, None]
        e = np.where(np.isnan(x64), 0, np.exp(x64 - m))
        z = e.sum(-1, keepdims=True)
        p = x64 - m - np.log(z)
        ent = np.where(e > 0, -(e / z) * p, 0).sum(-1)
    p[none], ent[none] = -np.inf, 0
    p[bad], ent[bad] = np.nan, np.nan
    order = np.stack([np.lexsort((np.arange(x.shape[1]), -np.where(np.isnan(r), 0, r).astype(np.float64), np.isnan(r)))[:top] for r in x]) if top else \
        np.zeros((len(x), 0), int)
    lp = np.where((ids >= 0) & (ids < x.shape[1]), np.take_along_axis(p, np.clip(ids, 0, x.shape[1] - 1), -1), np.where(bad, np.nan, -np.inf)[:, None])
    return lp, ent, order, np.take_along_axis(p, order, -1)


def run(x, ids, top, ld=None, entropy=True, ws=None):
    n, V = x.shape
    ld = ld or V
    m = ids.shape[1]
    big = np.full((n, ld), 1e30, F32)       # what lies between the rows is nobody's
    big[:, :V] = x
    b = [DevBuf.from_array(a) for a in (big, ids.astype(np.int32), np.full((n, max(m, 1)), 7.5, F32), np.full(n, 7.5, F32),
                                        np.full((n, max(top, 1)), -9, np.int32), np.full((n, max(top, 1)), 7.5, F32))]
    need = logprobs_ws(n, V, top)
    own = ws or DevBuf.from_array(np.zeros(need, np.uint8))
    logprobs_dev(b[0], ld, n, V, b[1] if m else 0, m, top, b[2] if m else 0, b[3] if entropy else 0, b[4] if top else 0, b[5] if top else 0,
                 own, need)
    sync()
    r = [b[2].download(F32, (n, m)), b[3].download(F32, (n,)), b[4].download(np.int32, (n, top)), b[5].download(F32, (n, top))]
    for t in b + ([] if ws else [own]):
        t.free()
    return r


def check(x, ids, top, got, entropy=True):
    lp, ent, order, tops = oracle(x, ids, top)
    # l - m is rounded (2^-24 of it), ln Z is off by its sum's rounding (2^-24 of each term, at most sqrt(V)/8 of
    # them a partial sum) and its own; the entropy's sum is of magnitude H
    V = x.shape[1]
    slack = 2.0 ** -24 * (4 + np.sqrt(V) / 8)
    assert (got[2] == order).all()
    for g, w in ((got[0], lp), (got[3], tops)):
        assert (np.isnan(g) == np.isnan(w)).all() and (np.isneginf(g) == np.isneginf(w)).all()
        f = np.isfinite(w)
        assert (np.abs(g[f] - w[f]) <= slack + 2.0 ** -22 * np.abs(w[f])).all(), np.abs(g[f] - w[f]).max()
    if entropy:
        assert (np.isnan(got[1]) == np.isnan(ent)).all()
        f = ~np.isnan(ent)
        assert (np.abs(got[1][f] - ent[f]) <= 4 * slack * (1 + np.abs(ent[f]))).all(), np.abs(got[1][f] - ent[f]).max()
    else:
        assert (got[1] == 7.5).all()


@pytest.mark.parametrize("n,V,m,top,spread,ld", [
    (1, 1, 1, 1, 1.0, None), (2, 2, 2, 2, 1.0, 3), (1, 64, 1, 64, 3.0, None), (3, 65, 2, 5, 1.0, 67), (5, 1000, 3, 20, 4.0, 1003),
    (1, 201088, 1, 20, 4.0, None), (2, 201089, 4, 64, 0.5, 201092), (7, 50257, 1, 5, 10.0, 50257), (64, 32000, 1, 0, 2.0, None),
    (4, 8191, 0, 20, 3.0, None), (3, 8192, 1, 1, 3.0, None), (3, 8193, 1, 32, 3.0, None), (300, 4097, 2, 7, 3.0, 4100),
    (2, 600000, 1, 40, 2.0, None), (33, 16384, 1, 64, 0.01, None)])
def test_logprobs(mh, n, V, m, top, spread, ld):
    say(f"logprobs n={n} V={V} m={m} top={top} spread={spread} ld={ld}")
    rng = np.random.default_rng(V + n)
    x = (rng.standard_normal((n, V)) * spread).astype(F32)
    ids = rng.integers(0, V, (n, m))
    check(x, ids, top, run(x, ids, top, ld))


@pytest.mark.parametrize("V", [37, 5000, 201088])
def test_ties_and_masks(mh, V):
    """All equal, a few values only, tokens masked by -inf and by the type's lowest value, zeros of both signs."""
    rng = np.random.default_rng(V)
    top = 20
    rows = [np.zeros(V), np.full(V, -3.4e38), rng.integers(0, 3, V), np.where(rng.random(V) < 0.9, -np.inf, rng.standard_normal(V)),
            np.where(rng.random(V) < 0.5, np.finfo(F32).min, rng.standard_normal(V) * 5), np.where(np.arange(V) == V - 1, 2.0, -np.inf),
            np.where(np.arange(V) % 2, 0.0, -0.0), -np.arange(V, dtype=float), np.arange(V, dtype=float),
            np.where(np.arange(V) < 25, 1.0, rng.standard_normal(V) * 0.01), rng.standard_normal(V) * 1e30]
    x = np.stack(rows).astype(F32)
    ids = np.stack([rng.integers(0, V, len(rows)), np.full(len(rows), -1), np.full(len(rows), V), np.full(len(rows), V - 1)], 1)
    say(f"logprobs ties and masks V={V}")
    check(x, ids, top, run(x, ids, top))


@pytest.mark.parametrize("V", [40, 9000])
def test_rows_without_a_distribution(mh, V):
    """Every token masked; NaN and +inf anywhere: each row by itself."""
    rng = np.random.default_rng(1)
    x = rng.standard_normal((6, V)).astype(F32)
    x[0] = -np.inf
    x[1, 3], x[2, V - 1], x[3] = np.nan, np.inf, np.nan
    x[4, ::2], x[4, 1] = np.nan, np.inf
    ids = rng.integers(0, V, (6, 3))
    say(f"logprobs rows without a distribution V={V}")
    check(x, ids, 20, run(x, ids, 20))


@pytest.mark.parametrize("kind", ["ascending", "descending", "equal", "masked", "nan", "few values", "nan then finite"])
def test_long_slices(mh, kind):
    """Rows that a block walks in many chunks: running lists that every chunk replaces, or none, or that are never full."""
    rng = np.random.default_rng(3)
    n, V, top = 64, 70001, 33
    x = np.empty((n, V), F32)
    if kind == "ascending":
        x[:] = np.arange(V) * 1e-3
    elif kind == "descending":
        x[:] = -np.arange(V) * 1e-3
    elif kind == "equal":
        x[:] = 1.5
    elif kind == "masked":
        x[:] = -np.inf
        x[:, ::5000] = rng.standard_normal((n, 15))
    elif kind == "nan":
        x[:] = np.nan
        x[1::2, 60000:60010] = 1.0
    elif kind == "nan then finite":
        x[:] = rng.standard_normal((n, V))
        x[:, :40000] = np.nan
    else:
        x[:] = rng.integers(0, 4, (n, V))
    ids = rng.integers(0, V, (n, 1))
    say(f"logprobs long slices {kind}")
    got = run(x, ids, top)
    rows = [0, 1, 40]
    check(x[rows], ids[rows], top, [g[rows] for g in got])
    assert all((g[2:] == g[:-2]).all() or np.isnan(g).any() or kind not in ("ascending", "descending", "equal") for g in got[1:])


def test_without_entropy(mh):
    rng = np.random.default_rng(1)
    x, ids = rng.standard_normal((3, 777)).astype(F32), rng.integers(0, 777, (3, 2))
    say("logprobs without entropy")
    check(x, ids, 3, run(x, ids, 3, entropy=False), entropy=False)


def test_overlaps_are_refused(mh):
    """Outputs and workspace over one another or over an input."""
    say("logprobs overlaps")
    n, V, m, top = 2, 500, 3, 4
    x, ids = DevBuf.from_array(np.zeros((n, V), F32)), DevBuf.from_array(np.zeros((n, m), np.int32))
    need = logprobs_ws(n, V, top)
    outs = [DevBuf.from_array(np.zeros(k, F32)) for k in (n * m, n, n * top, n * top, need // 4 + 1)]
    logprobs_dev(x, V, n, V, ids, m, top, *outs, need)
    for i in range(5):
        for other in [x, ids, *outs[:i], *outs[i + 1:]]:
            if i == 4 and other is not x:
                continue
            a = list(outs)
            a[i] = other
            with pytest.raises(MidgeHipError, match="overlap" if other.nbytes >= outs[i].nbytes else "overrun"):
                logprobs_dev(x, V, n, V, ids, m, top, *a, need)
    sync()
    for buf in (x, ids, *outs):
        buf.free()


def test_one_workspace_for_calls_in_order(mh):
    """Calls of other sizes one after another on one workspace, and the same bits again."""
    rng = np.random.default_rng(8)
    ws = DevBuf.from_array(np.zeros(max(logprobs_ws(9, 60000, 20), logprobs_ws(1, 201088, 64)), np.uint8))
    xs = [(rng.standard_normal(s) * 3).astype(F32) for s in ((9, 60000), (1, 201088), (2, 100))]
    first = {}
    for it in range(3):
        for i, (x, top) in enumerate(zip(xs, (20, 64, 7))):
            say(f"logprobs shared workspace round {it} call {i}")
            ids = np.full((x.shape[0], 1), 5)
            got = run(x, ids, top, ws=ws)
            check(x, ids, top, got)
            if i in first:
                assert all((a == b).all() for a, b in zip(first[i], got))
            first[i] = got
    ws.free()


def test_captured_and_replayed(mh):
    rng = np.random.default_rng(4)
    n, V, top = 3, 30000, 8
    say("logprobs captured")
    need = logprobs_ws(n, V, top)
    bufs = [DevBuf.from_array(a) for a in (np.zeros((n, V), F32), np.zeros((n, 1), np.int32), np.zeros((n, 1), F32), np.zeros(n, F32),
                                           np.zeros((n, top), np.int32), np.zeros((n, top), F32), np.zeros(need, np.uint8))]

    def call():
        logprobs_dev(bufs[0], V, n, V, bufs[1], 1, top, bufs[2], bufs[3], bufs[4], bufs[5], bufs[6], need)
    sync()
    st = Stream()
    g = Graph(st, call)
    for it in range(4):
        x, ids = (rng.standard_normal((n, V)) * 3).astype(F32), rng.integers(0, V, (n, 1))
        bufs[0].upload(x)
        bufs[1].upload(ids.astype(np.int32))
        g.launch(st)
        st.sync()
        read = lambda: [bufs[2].download(F32, (n, 1)), bufs[3].download(F32, (n,)), bufs[4].download(np.int32, (n, top)),     # noqa: E731
                        bufs[5].download(F32, (n, top))]
        got = read()
        check(x, ids, top, got)
        call()      # the program's own call between replays, on the same workspace
        sync()
        assert all((a == b).all() for a, b in zip(got, read()))
    for b in [*bufs, g, st]:
        b.free()


def test_a_workspace_for_the_largest_call(mh):
    """Calls of fewer rows on a workspace made for 33 rows; nothing behind it is written."""
    rng = np.random.default_rng(5)
    V, top, most = 32000, 20, 33
    need, room = logprobs_ws(most, V, top), 1 << 16
    ws = DevBuf.from_array(np.full(need + room, 0x5A, np.uint8))
    for n in (1, 5, 32, 33):
        say(f"logprobs on a workspace for {most} rows n={n}")
        x, ids = (rng.standard_normal((n, V)) * 3).astype(F32), rng.integers(0, V, (n, 1))
        b = [DevBuf.from_array(a) for a in (x, ids.astype(np.int32), np.zeros((n, 1), F32), np.zeros(n, F32), np.zeros((n, top), np.int32),
                                            np.zeros((n, top), F32))]
        logprobs_dev(b[0], V, n, V, b[1], 1, top, *b[2:], ws, need)
        sync()
        check(x, ids, top, [b[2].download(F32, (n, 1)), b[3].download(F32, (n,)), b[4].download(np.int32, (n, top)), b[5].download(F32, (n, top))])
        assert (ws.download(np.uint8, (need + room,))[need:] == 0x5A).all()
        for t in b:
            t.free()
    ws.free()


@pytest.mark.parametrize("V", [900, 4096, 70001])
def test_equal_rows_have_equal_results(mh, V):
    """Six kinds of rows in random order: each as the definition says, and the same bits in every equal row."""
    rng = np.random.default_rng(V)
    n, top = 96, 33
    base = np.stack([rng.standard_normal(V), np.full(V, 1.5), np.where(np.arange(V) % 50, -np.inf, rng.standard_normal(V)),
                     np.full(V, -np.inf), np.where(np.arange(V) == V // 2, np.nan, rng.standard_normal(V)), rng.integers(0, 4, V)]).astype(F32)
    which = rng.integers(0, len(base), n)
    which[:len(base)] = np.arange(len(base))
    ids = np.tile(rng.integers(0, V, (1, 2)), (n, 1))
    say(f"logprobs equal rows V={V}")
    got = run(base[which], ids, top)
    check(base, ids[:len(base)], top, [g[:len(base)] for g in got])
    for g in got:
        assert np.array_equal(g, g[:len(base)][which], equal_nan=g.dtype == F32)


@pytest.mark.parametrize("n,V,m,top", [(33001, 17, 1, 3), (3, 5000, 300, 2), (70000, 3, 0, 3)])
def test_many_rows_and_many_ids(mh, n, V, m, top):
    """More rows than a launch's second axis holds; more given tokens a row than a block has threads."""
    say(f"logprobs n={n} V={V} m={m} top={top}")
    rng = np.random.default_rng(n)
    x = (rng.standard_normal((n, V)) * 2).astype(F32)
    ids = rng.integers(-1, V + 1, (n, m))
    check(x, ids, top, run(x, ids, top))
