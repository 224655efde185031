"""mh_verify_dev on the GPU against its definition in 64 bits (tree_oracle):
trees and chains, drafts that were chosen or drawn, masked tokens, rows
without probabilities, ties; captured graphs; and a whole step of drafted
tokens through the cache. Decisions and tokens have to be equal: a draw lies
within 2^-50 of a border with a chance of 1e-9 over all the cases here."""
import numpy as np
import pytest

from conftest import say
from midge_amd import MidgeHipError, _lib, sync
from midge_amd import kv
from midge_amd.moe import Draft, verify_dev, verify_ws
from hip_graph import Graph, Stream
from kv_oracle import KV_F16, KV_MXFP4, Batch, KVRows, Pages
from test_gpu_kv import EPS, F32, Dev, tables, tolerance
from tree_oracle import SHAPES, tree, verify, weights

pytestmark = pytest.mark.gpu


class Drafts:
    """Sequences of `rows` rows each with logits whose drafts are likely ones; q: drafts drawn from a noisy copy."""

    def __init__(self, rows, V, shape, temp, drawn, rng, ld=0, ldq=0, spread=2.0, noise=0.7, front=0, behind=0, chain_null=False):
        self.rows, self.V, self.temp, self.chain_null = rows, V, temp, chain_null
        self.row0 = (front + np.concatenate(([0], np.cumsum(rows)))).astype(np.int32)
        n = int(self.row0[-1]) + behind
        self.ld, self.ldq, self.drawn = ld or V, ldq or V, drawn
        self.logits = np.full((n, self.ld), 1e9, F32)      # (behind a row's tokens: never looked at)
        self.logits[:, :V] = rng.standard_normal((n, V)) * spread
        self.q = np.full((n, self.ldq), 1e9, F32)
        heat = temp if temp > 0 else 1.0
        for r in range(n):
            self.q[r, :V] = weights(self.logits[r, :V] + (rng.standard_normal(V) * noise).astype(F32), heat)
        self.parent = np.full(n, -1, np.int32)
        self.token = rng.integers(0, V, n).astype(np.int32)
        self.u = rng.random(n).astype(F32)
        self.u[self.u >= 1] = 0.5
        for s, r in enumerate(rows):
            a = self.row0[s]
            self.parent[a:a + r] = tree(r, "chain" if chain_null else shape, rng)
            for i in range(1, r):
                p = self.q[a + max(self.parent[a + i], 0), :V].astype(np.float64)
                if drawn:
                    self.token[a + i] = rng.choice(V, p=p / p.sum())
                elif rng.random() < 0.9:
                    self.token[a + i] = np.argsort(-p)[min(V - 1, int(rng.integers(0, 3)))]

    def want(self):
        n_kept, kept, after = [], np.full((len(self.rows), max(max(self.rows), 1)), -1, np.int32), []
        for s, r in enumerate(self.rows):
            if r == 0:
                n_kept.append(0), after.append(-1)
                continue
            at = slice(self.row0[s], self.row0[s + 1])
            path, t = verify(self.logits[at, :self.V], [p if -1 <= p < i else -1 for i, p in enumerate(self.parent[at])], self.token[at], self.u[at], self.temp,
                             self.q[at, :self.V] if self.drawn else None)
            n_kept.append(len(path)), after.append(t)
            kept[s, :len(path)] = path
        return np.array(n_kept), kept, np.array(after)

    def device(self, dev, mis=0):
        """`mis`: floats by which the logits and q are off 16-byte alignment."""
        pad = lambda a: dev(np.concatenate((np.zeros(mis, F32), a.ravel()))).ptr + 4 * mis     # noqa: E731
        n = len(self.rows)
        self.out = [dev(np.full(m, 77, np.int32)) for m in (n + 1, n * max(max(self.rows), 1) + 1, n + 1)]
        self.bufs = dict(row0=dev(self.row0), parent=dev(self.parent), token=dev(self.token), u=dev(self.u), logits=pad(self.logits), q=pad(self.q))
        b = self.bufs
        self.draft = Draft(n, len(self.logits), max(max(self.rows), 1), b["row0"], 0 if self.chain_null else b["parent"], b["token"], b["u"], self.V,
                           b["logits"], self.ld, self.temp, b["q"] if self.drawn else 0, self.ldq)
        self.need = verify_ws(n, len(self.logits), self.V)
        self.ws = dev(np.full(self.need + 256, 0x5A, np.uint8))

    def run(self):
        verify_dev(self.draft, *self.out, self.ws, self.need)

    def got(self):
        n, w = len(self.rows), max(max(self.rows), 1)
        a, k, t = (o.download(np.int32, (m,)) for o, m in zip(self.out, (n + 1, n * w + 1, n + 1)))
        assert a[-1] == k[-1] == t[-1] == 77
        assert (self.ws.download(np.uint8, (self.need + 256,))[self.need:] == 0x5A).all()
        return a[:-1], k[:-1].reshape(n, w), t[:-1]

    def check(self, mis=0):
        dev = Dev()
        self.device(dev, mis)
        self.run()
        sync()
        got = self.got()
        dev.free()
        for name, g, w in zip(("n_kept", "kept", "next"), got, self.want()):
            assert (g == w).all(), (name, g, w)
        return got


@pytest.mark.parametrize("V", [1, 2, 7, 100, 1023, 1024, 1025, 5000, 33000])
@pytest.mark.parametrize("drawn", [0, 1])
@pytest.mark.parametrize("temp", [1.0, 0.25, 2.0, 0.0])
def test_verify(mh, V, drawn, temp):
    rng = np.random.default_rng(V * 10 + drawn)
    rows = [5, 1, 0, 9, 2, 3] if V > 10000 else [5, 1, 0, 64, 2, 33, 17, 1, 8]
    kept = 0
    for spread in (2.0, 6.0):
        for shape in SHAPES:
            say(f"verify V={V} drawn={drawn} temp={temp} spread={spread} {shape}")
            n_kept, _, _ = Drafts(rows, V, shape, temp, drawn, rng, ld=V + int(rng.integers(0, 5)), ldq=V + int(rng.integers(0, 5)), spread=spread,
                                  front=2, behind=3).check(int(rng.integers(0, 4)))
            kept += n_kept.sum()
        say(f"verify V={V} drawn={drawn} temp={temp} spread={spread} chains without parents")
        kept += Drafts(rows, V, "chain", temp, drawn, rng, spread=spread, chain_null=True).check()[0].sum()
    assert kept > 10 * len([r for r in rows if r])       # (rows beside the first ones: some drafts are kept)


@pytest.mark.parametrize("drawn", [0, 1])
def test_large_vocabulary(mh, drawn):
    for V, rows in ((201088, [8]), (201088, [3, 6, 1, 4]), (131072, [2, 2]), (262145, [4]), (3000001, [2])):
        for spread in (0.01, 2.0, 6.0) if V < 1000000 else (2.0,):
            say(f"verify V={V} drawn={drawn} spread={spread}")
            Drafts(rows, V, "any", 0.8, drawn, np.random.default_rng(V + drawn), spread=spread).check()


@pytest.mark.parametrize("drawn", [0, 1])
def test_many_refusals(mh, drawn):
    """Drafts that all follow one row and are nearly all refused: the same token again, tokens of no probability, and all
    tokens there are."""
    for V in (3, 40, 3000):
        for it in range(6):
            say(f"verify refusals V={V} drawn={drawn} {it}")
            rng = np.random.default_rng(it)
            d = Drafts([64, 30, 5], V, "wide", 1.0, drawn, rng, spread=3.0, noise=3.0)
            d.u[:] = 1 - rng.random(len(d.u)).astype(F32) ** 2 * 0.3      # large draws
            d.u = np.minimum(d.u, np.float32(1 - 2.0 ** -24)).astype(F32)
            if not drawn:
                d.token[:] = rng.permutation(np.arange(len(d.token)) % V)
            d.check()


@pytest.mark.parametrize("temp", [1.0, 0.0])
@pytest.mark.parametrize("drawn", [0, 1])
def test_masked_tokens_and_rows_without_probabilities(mh, temp, drawn):
    """-inf in most places, one token left, none left, NaN, +inf, the type's lowest and largest values; drafts outside the vocabulary."""
    for V in (50, 4000):
        for it in range(8):
            say(f"verify masked V={V} temp={temp} drawn={drawn} {it}")
            rng = np.random.default_rng(100 + it)
            d = Drafts([12] * 10, V, SHAPES[it % 4], temp, drawn, rng)
            for s in range(10):
                r = d.row0[s] + int(rng.integers(0, 4))
                x = d.logits[r]
                if s == 0:
                    x[rng.random(V) < 0.9] = -np.inf
                elif s == 1:
                    x[:] = -np.inf
                    x[it % V] = -3.0
                elif s == 2:
                    x[:] = -np.inf
                elif s == 3:
                    x[int(rng.integers(V))] = np.nan
                elif s == 4:
                    x[int(rng.integers(V))] = np.inf
                elif s == 5:
                    x[rng.random(V) < 0.5] = np.finfo(F32).min
                elif s == 6:
                    x[:] = np.finfo(F32).min
                elif s == 7:
                    x[::3] = np.finfo(F32).max
                elif s == 8:
                    d.token[d.row0[s] + 1:d.row0[s + 1]] = rng.choice([-1, V, -2 ** 31, 2 ** 31 - 1], 11)
                else:
                    x[:] = 0.25
                    x[::2] = -0.0
            d.check()


def test_ties_and_ends(mh):
    """Equal logits: the first maximum; draws of 0, of the largest below 1, and exactly on a border."""
    say("verify ties")
    d = Drafts([1] * 9, 4, "chain", 1.0, 0, np.random.default_rng(0))
    d.logits[:] = 1.5
    d.u[:] = [0, 0.25, np.nextafter(F32(0.25), F32(0)), 0.5, 0.75, 1 - 2.0 ** -24, 0.1, 0.9, 0.99]
    _, _, after = d.check()
    assert list(after[:6]) == [0, 1, 0, 2, 3, 3]
    d.temp = 0.0
    assert (d.check()[2] == 0).all()
    # a draft that has half of the probability, drawn on the border: u < p
    d = Drafts([2, 2], 2, "chain", 1.0, 0, np.random.default_rng(0))
    d.logits[:], d.token[:] = 0.0, 1
    d.u[:] = [0.3, 0.5, 0.3, np.nextafter(F32(0.5), F32(0))]
    n_kept, _, after = d.check()
    assert list(n_kept) == [1, 2] and after[0] == 0
    # drawn from the target itself: always kept
    d = Drafts([6, 20], 300, "any", 1.0, 1, np.random.default_rng(3), noise=0.0)
    d.check()


@pytest.mark.parametrize("drawn", [0, 1])
def test_values_that_are_no_draws_or_probabilities(mh, drawn):
    """NaN, negative and large u and q: some decision and a token of the vocabulary, no fault."""
    say(f"verify odd draws drawn={drawn}")
    rng = np.random.default_rng(8)
    d = Drafts([20] * 6, 700, "any", 1.0, drawn, rng)
    d.u[rng.random(len(d.u)) < 0.5] = np.nan
    d.u[rng.random(len(d.u)) < 0.2] = 1.5
    d.u[rng.random(len(d.u)) < 0.2] = -1.0
    d.q[rng.random(d.q.shape) < 0.1] = np.nan
    d.q[rng.random(d.q.shape) < 0.1] = -1.0
    dev = Dev()
    d.device(dev)
    d.run()
    sync()
    n_kept, kept, after = d.got()
    dev.free()
    assert ((n_kept >= 1) & (n_kept <= 20)).all() and ((after >= 0) & (after < 700)).all()
    for s in range(6):
        assert kept[s, 0] == 0 and (kept[s, n_kept[s]:] == -1).all() and (np.diff(kept[s, :n_kept[s]]) > 0).all()


def test_bad_sequences(mh):
    """Parents out of range count as none, sequences out of bounds keep nothing, and mh_sync says so."""
    rng = np.random.default_rng(12)
    for value in (1, 5, -2, 1 << 30):
        say(f"verify with a parent of {value}")
        d = Drafts([4, 4, 4], 90, "any", 1.0, 0, rng)
        d.parent[d.row0[1] + 1] = value
        dev = Dev()
        d.device(dev)
        d.run()
        with pytest.raises(MidgeHipError, match="out of bounds"):
            sync()
        sync()
        for g, w in zip(d.got(), d.want()):
            assert (g == w).all()
        dev.free()
    for ends in ([0, 4, 13, 12], [0, 9, 8, 12], [-1, 4, 8, 12], [0, 4, 4, 4 + (1 << 30)]):
        say(f"verify with rows at {ends}")
        d = Drafts([4, 4, 4], 90, "any", 1.0, 0, rng)
        good = d.want()
        d.row0[:] = ends
        dev = Dev()
        d.device(dev)
        d.run()
        with pytest.raises(MidgeHipError, match="out of bounds"):
            sync()
        got = d.got()
        dev.free()
        for s in range(3):
            if 0 <= ends[s] <= ends[s + 1] <= 12 and ends[s + 1] - ends[s] <= 4:
                if [ends[s], ends[s + 1]] == [4 * s, 4 * s + 4] and 0 <= ends[0] and ends[3] == 12:
                    assert all((g[s] == w[s]).all() for g, w in zip(got, good))
            else:
                assert got[0][s] == 0 and (got[1][s] == -1).all() and got[2][s] == -1


def test_no_rows(mh):
    say("verify of no rows")
    d = Drafts([0, 0], 10, "any", 1.0, 0, np.random.default_rng(0), behind=1)
    d.check()
    one = Drafts([1, 1, 1], 500, "any", 1.0, 0, np.random.default_rng(0))
    dev = Dev()
    one.device(dev)
    one.draft.c.row0 = None     # one row each
    one.run()
    sync()
    assert all((g == w).all() for g, w in zip(one.got(), one.want()))
    dev.free()


def test_many_sequences(mh):
    """Each sequence its own walk; the same bits from call to call."""
    for drawn in (0, 1):
        say(f"verify of 700 sequences drawn={drawn}")
        rng = np.random.default_rng(4)
        d = Drafts([int(r) for r in rng.integers(0, 7, 700)], 300, "any", 1.0, drawn, rng, front=1)
        d.check()


@pytest.mark.parametrize("drawn", [0, 1])
def test_captured_and_replayed(mh, drawn):
    """A captured call, replayed with other trees, tokens, draws and logits between the program's own calls; two graphs on two
    streams with a workspace each."""
    say(f"verify capture drawn={drawn}")
    rng, graphs, dev = np.random.default_rng(drawn), [], Dev()
    for temp in (0.7, 0.0):
        d = Drafts([6, 9, 1], 5000, "any", temp, drawn, rng)
        d.device(dev)
        sync()
        st = Stream()
        graphs.append((Graph(st, d.run), st, d))
    for it in range(4):
        for g, st, d in graphs:
            new = Drafts([[6, 9, 1], [1, 2, 9], [9, 5, 2], [3, 0, 9]][it], 5000, SHAPES[it], d.temp, drawn, rng, behind=[0, 4, 0, 4][it])
            for k in ("row0", "parent", "token", "u"):
                setattr(d, k, getattr(new, k))
                d.bufs[k].upload(getattr(new, k))
            d.rows, d.logits, d.q = new.rows, new.logits, new.q
            for k in ("logits", "q"):
                a = np.ascontiguousarray(getattr(new, k))
                _lib.call("mh_h2d", d.bufs[k], a.ctypes.data, a.nbytes)
        for g, st, d in graphs:         # both in flight
            g.launch(st)
        for g, st, d in graphs:
            st.sync()
        for g, st, d in graphs:
            got = [o.download(np.int32, (m,)) for o, m in zip(d.out, (3, 27, 3))]
            kept = np.full((3, 9), -1)
            n_kept, k, after = d.want()
            kept[:, :k.shape[1]] = k
            assert (got[0] == n_kept).all() and (got[1].reshape(3, 9) == kept).all() and (got[2] == after).all(), it
            d.run()
            sync()
            assert all((o.download(np.int32, (m,)) == g).all() for o, m, g in zip(d.out, (3, 27, 3), got))
    for g, st, d in graphs:
        g.free(), st.free()
    dev.free()


# ------------------------------------------------------------------ together

@pytest.mark.parametrize("dt", [KV_F16, KV_MXFP4])
@pytest.mark.parametrize("drawn", [0, 1])
@pytest.mark.parametrize("window", [0, 20])
@pytest.mark.parametrize("spread", [2, 6])
def test_steps_of_drafted_tokens(mh, dt, drawn, window, spread):
    """Some steps of a server that drafts: trees through append, attention, verification and keep on two layers' caches.
    After each the caches hold, bit for bit, what appending the kept tokens one by one would have put there, and the
    kept rows' attention is that of the tokens one by one."""
    say(f"drafted steps dt={dt} drawn={drawn} window={window} spread={spread}")
    rng, nh, nkv, hd, page, V, layers = np.random.default_rng(3 + drawn), 8, 2, 64, 16, 400, 2
    seqs, max_pages = [37, 5, 160], 20
    table = rng.permutation(64)[:60].reshape(3, 20).astype(np.int32)
    # what a token's projections and logits are, of any place: a fixed table each
    proj = [[rng.standard_normal((V, w * hd)).astype(F32) for w in (nh, nkv, nkv)] for _ in range(layers)]
    head = (rng.standard_normal((V, V)) * spread).astype(F32)
    co, si = tables(400, hd)
    # tree[layer] goes the drafted way, plain[layer] one token after the other
    start = [Pages(dt, nkv, hd, page, 64, rng) for _ in range(layers)]
    plain = [Pages(dt, nkv, hd, page, 64, rng) for _ in range(layers)]
    dev = Dev()
    dco, dsi = dev(co), dev(si)
    for a, b in zip(start, plain):
        for s, n in enumerate(seqs):
            a.fill(table[s], n, rng)
        a.upload()
        b.arr = [x.copy() for x in a.arr]
        b.upload()
    length, last = list(seqs), [int(t) for t in rng.integers(0, V, 3)]
    moved = 0
    for step in range(5 if spread == 2 else 9):
        d = Drafts([7, 4, 12], V, SHAPES[step % 3], 0.9, drawn, rng)
        n = len(d.token)
        d.token[d.row0[:-1]] = last
        for s in range(3):      # a row's logits are its token's; drafts from a noisy copy of its parent's
            for i in range(d.row0[s], d.row0[s + 1]):
                if i > d.row0[s]:
                    p = d.q[d.row0[s] + d.parent[i], :V].astype(np.float64)
                    d.token[i] = rng.choice(V, p=p / p.sum()) if drawn else int(np.argsort(-p)[rng.integers(0, 2)])
                d.logits[i] = head[d.token[i]]
                d.q[i] = weights((head[d.token[i]] + rng.standard_normal(V) * 0.5).astype(F32), 0.9)
        d.device(dev)
        b = Batch([(m + r, r) for m, r in zip(length, d.rows)], page, rng, n_pages=64, max_pages=max_pages)
        b.pages[:] = table
        b.upload()
        outs = []
        for l in range(layers):
            q, k, v = (dev(x[d.token]) for x in proj[l])
            qo, out = dev(np.zeros((n, nh * hd), F32)), dev(np.zeros((n, nh * hd), F32))
            kv.tree_append_dev(start[l].cache, b.batch, d.bufs["parent"], KVRows(nh, 400, EPS, q, k, v, nh * hd, nkv * hd, nkv * hd, qo,
                                                                                rope_cos=dco, rope_sin=dsi))
            need = kv.tree_attention_ws(start[l].cache, b.batch, nh)
            kv.tree_attention_dev(start[l].cache, b.batch, d.bufs["parent"], nh, qo, out, dev(np.zeros(need, np.uint8)), need, 0.125, window)
            outs.append(out)
        d.run()
        ln = dev(np.zeros(3, np.int32))
        kv.keep_dev([p.cache for p in start], b.batch, d.out[0], d.out[1], ln)
        sync()
        n_kept, kept, after = d.got()
        for g, w in zip((n_kept, kept, after), d.want()):
            assert (g == w).all()
        assert (ln.download(np.int32, (3,)) == np.array(length) + n_kept).all()
        # the kept tokens one by one
        for j in range(int(n_kept.max())):
            some = [s for s in range(3) if j < n_kept[s]]
            one = Batch([(length[s] + j + 1, 1) for s in some], page, rng, n_pages=64, max_pages=max_pages, one=True)
            one.pages[:] = table[some]
            one.upload()
            tokens = [int(d.token[d.row0[s] + kept[s, j]]) for s in some]
            for l in range(layers):
                q, k, v = (dev(x[tokens]) for x in proj[l])
                qo, out = dev(np.zeros((len(some), nh * hd), F32)), dev(np.zeros((len(some), nh * hd), F32))
                kv.append_dev(plain[l].cache, one.batch, KVRows(nh, 400, EPS, q, k, v, nh * hd, nkv * hd, nkv * hd, qo, rope_cos=dco, rope_sin=dsi))
                need = kv.attention_ws(plain[l].cache, one.batch, nh)
                kv.attention_dev(plain[l].cache, one.batch, nh, qo, out, dev(np.zeros(need, np.uint8)), need, 0.125, window)
                sync()
                got, want = outs[l].download(F32, (n, nh * hd)), out.download(F32, (len(some), nh * hd))
                for i, s in enumerate(some):
                    # both are within tolerance() of the formula; scores of q and k of at most 8 deviations of hd terms
                    assert np.abs(got[d.row0[s] + kept[s, j]] - want[i]).max() <= 2 * tolerance(0.125 * 8 * hd, 8.0, length[s] + j + 1), (step, j, s)
            one.free()
        moved += sum(int((kept[s, :n_kept[s]] != np.arange(n_kept[s])).any()) for s in range(3))
        for s in range(3):
            length[s] += int(n_kept[s])
            last[s] = int(after[s])
        for l in range(layers):
            a, c = start[l].download(), plain[l].download()
            for s in range(3):
                for w in (0, 1):
                    x, y = (p.tokens(table[s], length[s], w, m) for p, m in ((start[l], a), (plain[l], c)))
                    assert (x == y).all(), (step, l, s, w)
        b.free()
    if spread > 2:
        assert moved > 0 and sum(length) > sum(seqs) + 27       # drafts were kept, and rows moved
    dev.free(*start, *plain)
