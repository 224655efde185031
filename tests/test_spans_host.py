"""Rows that lie far apart, without a GPU: the bytes from the first to the end
of the last pass 64 bits and look like few. Such a call is refused by its
arguments alone; the largest spans that can be counted are not."""
import ctypes as C

import pytest

from midge_amd import _lib
from test_kv_host import A, ARG, NOINIT, append, batch, cache, rows
from test_tree_host import append as tree_append, check_draft

FAR = 1 << 40       # floats between two rows, at most
# (rows, stride) whose span is 2^64 bytes and a row's, several times that and a row's, and just past 2^63
WRAP = [((1 << 22) + 1, FAR), ((1 << 23) + 1, FAR), ((1 << 23) + 1, FAR >> 1), ((1 << 21) + 1, FAR)]
far = pytest.mark.parametrize("n,ld", WRAP)


def logprobs(n, ld):
    return _lib.load().mh_logprobs_dev(1 << 20, ld, n, 100, None, 0, 0, None, A, None, None, 1 << 32, 1 << 40)


@far
def test_rows_whose_span_passes_64_bits(n, ld):
    assert ((n - 1) * ld * 4) % (1 << 64) in (0, 1 << 63)
    for which in ("ldq", "ldk", "ldv"):
        r = rows(q_out=1 << 44, **{which: ld})
        assert append(cache(), batch(n_rows=n), r) == ARG
        assert tree_append(cache(), batch(n_rows=n), r, parent=8 * A) == ARG
    assert check_draft(n_rows=n, ld=ld, q=0, ldq=0, logits=1 << 44, token=1 << 50, u=1 << 51, parent=1 << 52) == ARG
    assert check_draft(n_rows=n, ldq=ld, logits=1 << 44, q=1 << 53, token=1 << 50, u=1 << 51, parent=1 << 52) == ARG
    assert logprobs(n, ld) == ARG


def test_one_row_lies_any_distance_from_the_next():
    if _lib.load().mh_sync() != NOINIT:
        pytest.skip("the library is initialised")
    one = dict(n_seqs=1, n_rows=1, row0=0)
    assert check_draft(**one, ld=FAR, ldq=FAR) == NOINIT
    assert append(cache(), batch(**one), rows(ldq=FAR, ldk=FAR, ldv=FAR)) == NOINIT
    assert logprobs(1, FAR) == NOINIT
    assert logprobs(0, FAR) == NOINIT
