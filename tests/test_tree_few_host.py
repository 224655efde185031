"""That the cases of test_gpu_kvtree_few are the ones that its kernel is chosen
for: the workspace of the kernel for few columns is its plan and two partial
results of 64 columns for each of 1024 blocks, and no other's."""
import ctypes as C

import pytest

from test_gpu_kvtree_few import CASES, ODD, heads_of
from test_kv_host import A, batch, cache, rc


def ws(dt, nkv, hd, g, seqs, rows, most, name="mh_kv_tree_attention_ws"):
    n = C.c_uint64()
    assert rc(name, C.byref(cache(dt=dt, n_kv_heads=nkv, head_dim=hd).c), C.byref(batch(n_seqs=seqs, n_rows=rows, max_rows=most, row0=A).c), nkv * g,
              C.byref(n)) == 0
    return n.value


def few(hd, seqs):
    return (8 * (seqs + 1) + 15) // 16 * 16 + 2 * 1024 * 64 * (hd + 2) * 4


@pytest.mark.parametrize("dt,hd,g,r,n", sorted({c[:5] for c in CASES} | {(*c, 1) for c in ODD}))
def test_cases_take_the_kernel_for_few_columns(dt, hd, g, r, n):
    assert 48 < g * r <= 64
    for nkv in {2, heads_of(g, hd)}:
        rows = 2 * r * n + 1
        assert ws(dt, nkv, hd, g, n, rows, r) == few(hd, n)
        # neither chunks nor five trees nor one more row do
        assert ws(dt, nkv, hd, g, n, rows, r, "mh_kv_attention_ws") != few(hd, n)
        assert ws(dt, nkv, hd, g, 5, rows, r) != few(hd, 5)
        assert g * (r + 1) <= 64 or r == 64 or ws(dt, nkv, hd, g, n, rows, r + 1) != few(hd, n)


def test_every_width_and_number_of_sequences_is_among_them():
    assert {(c[0], c[1], c[4]) for c in CASES} == {(dt, hd, n) for dt in (0, 1) for hd in (32, 64, 96, 128) for n in (1, 2, 4)}
    for dt in (0, 1):
        for hd in (32, 64, 96, 128):
            assert {c[2] * c[3] for c in CASES if c[:2] == (dt, hd)} >= {49, 52, 56, 62, 64}
