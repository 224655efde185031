"""Trees of drafted tokens without a GPU: refused arguments, mh_kv_tree_check
on host batches, and what the verification's definition promises."""
import ctypes as C

import numpy as np
import pytest

from midge_amd import _lib
from midge_amd.kv import KV_F16, KV_MXFP4, KVBatch, tree_check
from midge_amd.moe import Draft
from test_kv_host import A, ARG, DTYPE, NOINIT, RANGE, UNSUP, batch, cache, rc, rows
from tree_oracle import paths, seen, tree, verify, weights


def append(c=None, b=None, r=None, parent=A):
    return rc("mh_kv_tree_append_dev", C.byref((c or cache()).c), C.byref((b or batch()).c), parent, C.byref((r or rows()).c))


def attend(c=None, b=None, parent=2 * A, nh=4, window=0, scale=0.125, q=A, out=1 << 20, ws=1 << 32, n=1 << 40, sink=None):
    return rc("mh_kv_tree_attention_dev", C.byref((c or cache()).c), C.byref((b or batch()).c), parent, nh, window, scale, sink, q, out, ws, n)


def keep(caches=None, b=None, n_kept=A, kept=2 * A, len_out=3 * A, n=None):
    cs = caches or [cache(k=1 << 24, v=1 << 25, ks=1 << 26, vs=1 << 27)]
    a = (_lib.MhKvCache * len(cs))(*[c.c for c in cs])
    return rc("mh_kv_keep_dev", a, len(cs) if n is None else n, C.byref((b or batch(row0=4 * A, len=5 * A, pages=6 * A)).c), n_kept, kept, len_out)


@pytest.mark.parametrize("kw,code", [
    (dict(dt=2), DTYPE), (dict(head_dim=48), UNSUP), (dict(n_kv_heads=0), ARG), (dict(page=48), ARG), (dict(n_pages=0), ARG), (dict(k=0), ARG),
    (dict(ks=0), ARG), (dict(v=A + 8), ARG)])
def test_cache_refusals(kw, code):
    c = cache(**kw)
    assert append(c=c) == code and attend(c=c) == code and keep([c]) == code
    assert rc("mh_kv_tree_attention_ws", C.byref(c.c), C.byref(batch().c), 4, C.byref(C.c_uint64())) == code


@pytest.mark.parametrize("kw,code", [
    (dict(n_seqs=0), ARG), (dict(n_rows=-1), ARG), (dict(max_rows=0), ARG), (dict(max_pages=0), ARG), (dict(len=0), ARG), (dict(row0=0), ARG),
    (dict(max_rows=65), UNSUP)])
def test_batch_refusals(kw, code):
    b = batch(**kw)
    assert append(b=b) == code and attend(b=b) == code
    assert keep(b=batch(**{**dict(row0=4 * A, len=5 * A, pages=6 * A), **kw})) == code
    if kw != dict(row0=0):
        assert rc("mh_kv_tree_attention_ws", C.byref(cache().c), C.byref(b.c), 4, C.byref(C.c_uint64())) == code


def test_tree_refusals():
    for kw in (dict(parent=0), dict(parent=A + 2)):
        assert append(**kw) == ARG and attend(**kw) == ARG
    assert append(parent=1 << 20) == ARG and append(parent=(1 << 20) + 5 * 1024 - 4) == ARG         # under q_out
    assert attend(parent=1 << 20) == ARG and attend(parent=(1 << 32) + 16) == ARG                   # under out, the workspace
    for kw in (dict(nh=3), dict(window=-1), dict(scale=float("nan")), dict(q=0), dict(ws=0), dict(n=0), dict(out=A + 4), dict(ws=A), dict(sink=1 << 20)):
        assert attend(**kw) == ARG, kw
    assert append(r=rows(q=0)) == ARG and append(r=rows(q_out=2 * A)) == ARG
    lib = _lib.load()
    for args in ((None, C.byref(batch().c)), (C.byref(cache().c), None)):
        assert lib.mh_kv_tree_append_dev(*args, A, C.byref(rows().c)) == ARG
        assert lib.mh_kv_tree_attention_dev(*args, A, 4, 0, 1.0, None, A, 1 << 20, 1 << 32, 1 << 40) == ARG
    assert lib.mh_kv_tree_append_dev(C.byref(cache().c), C.byref(batch().c), A, None) == ARG
    assert lib.mh_kv_tree_attention_ws(C.byref(cache().c), C.byref(batch().c), 4, None) == ARG


def test_keep_refusals():
    big = [cache(k=(1 << 24) + i * 0x10000, v=(1 << 25) + i * 0x10000, ks=(1 << 26) + i * 0x10000, vs=(1 << 27) + i * 0x10000) for i in range(3)]
    size = 9 * 2 * 16 * 64 // 2
    for kw in (dict(n_kept=0), dict(kept=0), dict(len_out=0), dict(n_kept=A + 1), dict(kept=A + 2), dict(len_out=A + 3), dict(n=0), dict(n=-1), dict(n=4097)):
        assert keep(big, **kw) == ARG, kw
    # another type or shape than the first; one cache twice; parts of two in one place
    for kw in (dict(dt=KV_F16), dict(n_kv_heads=3), dict(head_dim=32), dict(page=32), dict(n_pages=8), dict(k=1 << 24), dict(v=1 << 24),
               dict(k=(1 << 24) + size - 16), dict(ks=1 << 26), dict(vs=(1 << 26) + size // 16 - 16), dict(ks=(1 << 24))):
        other = cache(**{**dict(k=1 << 28, v=1 << 29, ks=1 << 30, vs=1 << 31), **kw})
        assert keep([big[0], other]) == ARG, kw
    assert keep([big[0], big[1], big[0]]) == ARG
    # what is written over what is read
    for at in (A, A + 4, 2 * A, 2 * A + 16, 4 * A + 8, 5 * A, 6 * A + 20, 1 << 24, (1 << 25) + size - 4):
        assert keep(big, len_out=at) == ARG, at
    for kw in (dict(n_kept=1 << 24), dict(kept=(1 << 26) + 16)):
        assert keep(big, **kw) == ARG, kw
    assert rc("mh_kv_keep_dev", None, 1, C.byref(batch().c), A, A, A) == ARG
    assert rc("mh_kv_keep_dev", (_lib.MhKvCache * 1)(big[0].c), 1, None, A, 2 * A, 3 * A) == ARG


def draft(**kw):
    d = dict(n_seqs=2, n_rows=5, max_rows=4, row0=A, parent=2 * A, token=3 * A, u=4 * A, vocab=100, logits=1 << 20, ld=100, temp=1.0, q=1 << 22, ldq=128)
    return Draft(**{**d, **kw})


def check_draft(n_kept=5 * A, kept=6 * A, next=7 * A, ws=1 << 32, nb=1 << 40, **kw):
    return rc("mh_verify_dev", C.byref(draft(**kw).c), n_kept, kept, next, ws, nb)


def test_verify_refusals():
    for kw in (dict(n_seqs=0), dict(n_rows=-1), dict(n_rows=1 << 24), dict(max_rows=0), dict(row0=0), dict(token=0), dict(u=0), dict(logits=0), dict(vocab=0),
               dict(vocab=(1 << 30) + 1, ld=1 << 31), dict(ld=99), dict(ldq=99), dict(ld=1 << 41), dict(temp=float("nan")), dict(temp=float("inf")),
               dict(n_kept=0), dict(kept=0), dict(next=0), dict(ws=0), dict(nb=0), dict(ws=(1 << 32) + 8), dict(logits=(1 << 20) + 2), dict(q=(1 << 22) + 1),
               dict(token=A + 2), dict(parent=A + 1), dict(u=A + 3), dict(next=A + 1),
               # outputs over each other and over inputs
               dict(n_kept=6 * A), dict(next=6 * A + 28), dict(kept=7 * A), dict(kept=A), dict(next=2 * A + 16), dict(n_kept=3 * A), dict(next=4 * A),
               dict(kept=1 << 20), dict(next=(1 << 22) + 4 * (4 * 128 + 99)), dict(ws=1 << 20), dict(ws=1 << 22)):
        assert check_draft(**kw) == ARG, kw
    assert check_draft(max_rows=65) == UNSUP
    assert rc("mh_verify_dev", None, A, A, A, A, 1 << 40) == ARG
    assert rc("mh_verify_ws", 2, 5, 100, None) == ARG and rc("mh_verify_ws", 0, 5, 100, C.byref(C.c_uint64())) == ARG


def test_calls_before_init():
    if _lib.load().mh_sync() != NOINIT:
        pytest.skip("the library is initialised")
    assert append() == NOINIT and attend() == NOINIT and keep() == NOINIT and check_draft() == NOINIT
    # no draft's probabilities; the last floats of one row beside the next thing
    assert check_draft(q=0, ldq=0) == NOINIT and check_draft(next=(1 << 22) + 4 * (4 * 128 + 100)) == NOINIT and check_draft(temp=0.0) == NOINIT


def test_verify_workspace_of_the_largest_call():
    def ws(n, v):
        b = C.c_uint64()
        assert rc("mh_verify_ws", 1, n, v, C.byref(b)) == 0
        return b.value
    ns, vs = [0, 1, 2, 7, 63, 64, 1000, (1 << 24) - 1], [1, 100, 1023, 1024, 1025, 32000, 201088, 262144, 262145, 1 << 30]
    for n in ns:
        sizes = [ws(n, v) for v in vs]
        assert all(a <= b for a, b in zip(sizes, sizes[1:]))
    for v in vs:
        sizes = [ws(n, v) for n in ns]
        assert all(a <= b for a, b in zip(sizes, sizes[1:]))


@pytest.mark.parametrize("kw,bad", [
    ({}, None), (dict(row0=(3, 8)), 2), (dict(len=(0, 49)), 0), (dict(len=(0, 2)), 0), (dict(len=(2, 3)), 2), (dict(pages=((0, 0), -1)), 0),
    (dict(parent=(0, 0)), 0), (dict(parent=(2, -2)), 0), (dict(parent=(5, 3)), 2), (dict(parent=(5, 2)), 2), (dict(parent=(5, 1)), None), (dict(parent=(4, 0)), None)])
def test_check(kw, bad):
    row0, ln = np.array([0, 3, 3, 7], np.int32), np.array([33, 0, 16], np.int32)
    pages, parent = np.array([[8, 0, 3], [-1, -1, -1], [5, -1, -1]], np.int32), np.array([-1, 0, 0, -1, -1, 0, 2], np.int32)
    for k, v in kw.items():
        {"row0": row0, "len": ln, "pages": pages, "parent": parent}[k].__setitem__(*v)
    b = KVBatch(3, 7, 4, 3, row0.ctypes.data, ln.ctypes.data, pages.ctypes.data)
    if bad is None:
        tree_check(cache(), b, parent.ctypes.data)
        return
    with pytest.raises(_lib.MidgeHipError, match=f"sequence {bad}:") as e:
        tree_check(cache(), b, parent.ctypes.data)
    assert e.value.code == RANGE


@pytest.mark.parametrize("dt", [KV_F16, KV_MXFP4])
@pytest.mark.parametrize("hd,nkv,group", [(64, 8, 8), (128, 4, 8), (128, 8, 4), (256, 1, 8), (32, 3, 5), (96, 1, 64), (192, 2, 1)])
def test_attention_workspace_of_the_largest_batch(dt, hd, nkv, group):
    """A workspace for the most sequences, rows and rows a sequence serves every smaller batch of trees."""
    c = cache(dt=dt, head_dim=hd, n_kv_heads=nkv)

    def ws(seqs, rows, most, row0=A):
        size = C.c_uint64()
        assert rc("mh_kv_tree_attention_ws", C.byref(c.c), C.byref(batch(n_seqs=seqs, n_rows=rows, max_rows=most, row0=row0).c), nkv * group,
                  C.byref(size)) == 0
        return size.value
    seqs, mosts = [1, 2, 3, 4, 5, 8, 31, 64, 257, 1000], [*range(1, 18), 31, 32, 33, 48, 63, 64]
    for i, s in enumerate(seqs):
        for rows in (s, s + 5, 64, 513, 5000):
            sizes = [ws(s, rows, m) for m in mosts]
            assert all(a <= b for a, b in zip(sizes, sizes[1:])), (s, rows)
            for m, size in zip(mosts, sizes):
                assert ws(s, rows + 1, m) >= size and (i == 0 or ws(seqs[i - 1], rows, m) <= size)
                assert rows != s or ws(s, s, 1, 0) <= size


def test_keep_of_no_caches():
    from midge_amd.kv import keep_dev
    with pytest.raises(_lib.MidgeHipError, match="0 caches") as e:
        keep_dev([], batch(), A, A, A)
    assert e.value.code == ARG


# ------------------------------------------------------------ definitions

def test_paths_and_what_they_see():
    p = paths([-1, 0, 0, 1, -1, 3, 2])
    assert p == [[0], [0, 1], [0, 2], [0, 1, 3], [4], [0, 1, 3, 5], [0, 2, 6]]
    assert seen(5, p[5], 0) == [0, 1, 2, 3, 4, 5, 6, 8, 10]
    assert seen(5, p[5], 6) == [3, 4, 5, 6, 8, 10] and seen(5, p[5], 2) == [8, 10] and seen(5, p[4], 1) == [9] and seen(0, p[4], 3) == [4]
    assert tree(4, "chain", None) == [-1, 0, 1, 2]


@pytest.mark.parametrize("drawn", [0, 1])
@pytest.mark.parametrize("parent", [[-1, 0], [-1, 0, 0, 0], [-1, 0, 1], [-1, 0, 0, 1]])
def test_verified_tokens_follow_the_target(drawn, parent):
    """What verify() gives as the first new token is distributed as the target alone would have it: frequencies of N
    independent runs, each within 5 standard deviations of its probability (12 tokens, 8 settings: 1 in 20000 by chance)."""
    rng = np.random.default_rng(5 + drawn + len(parent))
    V, N, temp = 12, 20000, 0.7
    logits = (rng.standard_normal((len(parent), V)) * 1.5).astype(np.float32)
    q = np.array([weights((x + rng.standard_normal(V)).astype(np.float32), temp) for x in logits])
    count = np.zeros(V)
    for _ in range(N):
        token = [0] * len(parent)
        for i in range(1, len(parent)):
            # drawn from q, or chosen without regard to the draws: the likeliest few under q
            token[i] = rng.choice(V, p=q[parent[i]]) if drawn else int(np.argsort(-q[parent[i]])[i % 3])
        path, after = verify(logits, parent, token, rng.random(len(parent)), temp, q if drawn else None)
        count[token[path[1]] if len(path) > 1 else after] += 1
    p = weights(logits[0], temp)
    assert (np.abs(count / N - p) <= 5 * np.sqrt(p * (1 - p) / N) + 1 / N).all()


def test_refused_siblings_in_one_step():
    """max(max(p - a q, 0) / W - q, 0) is max(p - (a + W) q, 0) / W: the residual after several refusals."""
    rng = np.random.default_rng(1)
    p, q = rng.dirichlet(np.ones(50)), rng.dirichlet(np.ones(50))
    step, a, w = p.copy(), 0.0, 1.0
    for _ in range(6):
        rest = np.maximum(step - q, 0.0)
        step = rest / rest.sum()
        a += w
        w = np.maximum(p - a * q, 0.0).sum()
        assert np.allclose(step, np.maximum(p - a * q, 0.0) / w, rtol=1e-9, atol=1e-15)
