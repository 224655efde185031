"""mh_verify_dev called as its header allows and no list of cases has it:
drafts refused until rounding leaves nothing, rows named by sequences out of
order or by two of them, calls that take turns on one workspace, grids cut in
two. A row's sums are within 2^-45 of its whole sum, whatever their order: a
draw lies that near a border with a chance of 1e-8 over all the cases here."""
import numpy as np
import pytest

from conftest import say
from midge_amd import MidgeHipError, sync
from test_gpu_kv import F32, Dev
from test_gpu_verify import Drafts
from tree_oracle import verify

pytestmark = pytest.mark.gpu


def test_masked_drafts_after_all_others_are_refused(mh):
    """Three drafts take a row's probabilities but for what rounding leaves, each refused by the largest draw; the two
    after them are masked: neither is kept, and the token after is not one of them."""
    n = 400
    say(f"verify, masked drafts behind {n} rows that hold nothing else")
    rng = np.random.default_rng(7)
    d = Drafts([6] * n, 5, "wide", 1.0, 0, rng)
    d.logits[:] = -np.inf
    for s in range(n):      # weights of about 1, 2^-23 and 2^-46
        d.logits[6 * s, :3] = [0.0, -np.log(2.0) * (22.5 + rng.random()), -np.log(2.0) * (45.5 + rng.random())]
        d.token[6 * s + 1:6 * s + 6] = [0, 1, 2, 3, 4]
    d.u[:] = F32(1 - 2.0 ** -24)
    dev = Dev()
    d.device(dev)
    d.run()
    sync()
    n_kept, kept, after = d.got()
    dev.free()
    refused = 0
    for s in range(n):
        assert not set(kept[s, :n_kept[s]]) & {4, 5}, s
        refused += n_kept[s] == 1
        # (a kept draft's own row has no token)
        assert after[s] == -1 if n_kept[s] > 1 else 0 <= after[s] < 3, s
    assert refused > n // 10        # some rows had all three refused, so that the masked ones were tried


def out_of_order(d, ends, most):
    """Run with row0 = ends on arrays of d; each sequence whose own rows are in bounds has the definition's result."""
    d.row0 = np.array(ends, np.int32)
    d.rows = [most] * (len(ends) - 1)     # (max_rows, and the outputs' width)
    dev = Dev()
    d.device(dev)
    for _ in range(3):
        d.run()
        with pytest.raises(MidgeHipError, match="out of bounds"):
            sync()
        n_kept, kept, after = d.got()
        for s, (a, b) in enumerate(zip(ends, ends[1:])):
            if 0 <= a < b <= len(d.logits) and b - a <= most:
                path, t = verify(d.logits[a:b, :d.V], d.parent[a:b], d.token[a:b], d.u[a:b], d.temp, d.q[a:b, :d.V] if d.drawn else None)
            else:
                path, t = [], -1
            assert list(kept[s]) == path + [-1] * (most - len(path)) and n_kept[s] == len(path) and after[s] == t, (s, path, t, kept[s], after[s])
    dev.free()


@pytest.mark.parametrize("drawn", [0, 1])
@pytest.mark.parametrize("temp", [1.0, 0.0])
@pytest.mark.parametrize("ends", [[4, 0, 4, 8], [0, 4, 8, 2], [8, 12, 0, 4], [6, 2, 6, 12], [0, 4, 0, 4]])
def test_sequences_out_of_order(mh, ends, temp, drawn):
    """Row ranges that do not ascend: those in bounds are looked at, the others are reported."""
    for V in (90, 5000):
        say(f"verify, sequences at {ends} V={V} temp={temp} drawn={drawn}")
        rng = np.random.default_rng(V)
        # (a sequence's rows are the same tree wherever the ranges begin: all follow row 0, in a row of their own)
        d = Drafts([12], V, "wide", temp, drawn, rng, spread=4.0, noise=2.0)
        d.parent[:] = -1
        for a, b in zip(ends, ends[1:]):
            d.parent[a + 1:b] = 0
        out_of_order(d, ends, 6)


@pytest.mark.parametrize("temp", [1.0, 0.0])
@pytest.mark.parametrize("drawn", [0, 1])
def test_sequences_that_share_rows(mh, drawn, temp):
    """Two sequences that name the same rows, each from a place of its own: drafts of drawn ones are refused in both, and
    both walk on with their own rows' places."""
    for V, it in [(300, i) for i in range(10)] + [(5000, 10), (9000, 11)]:
        say(f"verify, shared rows V={V} temp={temp} drawn={drawn} {it}")
        rng = np.random.default_rng(it)
        d = Drafts([12], V, "wide", temp, drawn, rng, spread=4.0, noise=2.0)
        d.parent[:] = [-1, 0, 0, 0, -1, 0, 0, 0, 1, 2, 0, 3]        # (of rows 0 .. 8 and of 4 .. 12)
        d.u[1:4] = 0.99                                             # (the first sequence comes to rows 5 .. 7)
        for i in (5, 6, 7):     # likely tokens after the one first row or the other
            d.token[i] = int(np.argsort(-d.logits[(0, 4)[int(rng.integers(2))], :V])[rng.integers(0, 3)])
        out_of_order(d, [0, 8, 4, 12], 8)


@pytest.mark.parametrize("drawn", [0, 1])
def test_calls_that_take_turns_on_one_workspace(mh, drawn):
    """Calls of several sizes in turn, each with its own outputs every time: nothing of a call before is found (counters,
    sums, rows), and which block of a sequence ends last makes no difference."""
    dev, ws, need, ds = Dev(), None, 0, []
    for V, rows, shape in ((40000, [9, 1, 17, 5], "wide"), (300, [int(r) for r in np.random.default_rng(1).integers(0, 7, 700)], "any"),
                           (9001, [64, 3], "roots"), (40000, [6] * 8, "chain")):
        d = Drafts(rows, V, shape, 1.0, drawn, np.random.default_rng(V + len(rows)), spread=3.0, noise=2.0, chain_null=shape == "chain")
        d.device(dev)
        need = max(need, d.need)
        ds.append((d, d.want()))
    ws = dev(np.full(need, 0x5A, np.uint8))
    for d, _ in ds:
        d.ws, d.need = ws, need
    for it in range(8):
        for k in range(len(ds)):
            i = (k * (1 + it % 3) + it) % len(ds)
            d, want = ds[i]
            say(f"verify in turn drawn={drawn} pass {it} call {i}")
            for o in d.out:
                o.upload(np.full(o.nbytes // 4, 77, np.int32))
            d.run()
            n, w = len(d.rows), max(max(d.rows), 1)
            sync()
            got = [o.download(np.int32, (m,))[:-1] for o, m in zip(d.out, (n + 1, n * w + 1, n + 1))]
            assert all((g == x.ravel()).all() for g, x in zip(got, want)), (it, i)
    dev.free()


@pytest.mark.parametrize("drawn", [0, 1])
def test_more_rows_and_sequences_than_a_grid_holds(mh, drawn):
    """49500 rows of 33000 sequences: the launches over rows and over waiting sequences are two each."""
    say(f"verify of 33000 sequences drawn={drawn}")
    d = Drafts([1 + s % 2 for s in range(33000)], 24, "any", 1.0, drawn, np.random.default_rng(5), spread=1.0, noise=2.0)
    d.check()
