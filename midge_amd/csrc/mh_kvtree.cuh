// mh_kvtree.cuh — trees of drafted tokens among a sequence's rows
// (mh_kv_tree_*, mh_kv_keep_dev): bounds, and the paths from a tree's first
// rows to its others.
#pragma once

#include "mh_kv.cuh"
#include "mh_xchg.cuh"

namespace mh {

// Rows of a sequence: a wave holds one a lane, and the rows on a path are
// bits of a word.
constexpr int kTreeRows = 64;

// kv_seq for trees: the rows lie behind base >= 0 cached tokens.
__host__ __device__ inline bool kv_tree_seq(const KvBatchDev &b, int shift, int s, KvSeq *q) {
    return kv_seq(b, shift, s, q) && q->len >= q->n && q->n <= kTreeRows;
}
template <bool TREE>
__host__ __device__ inline bool kv_rows_of(const KvBatchDev &b, int shift, int s, KvSeq *q) {
    return TREE ? kv_tree_seq(b, shift, s, q) : kv_seq(b, shift, s, q);
}

// Host side (mh_kvtree.hip): the arguments that every function on trees has.
int kv_tree_validate(const mh_kv_batch *b, const int32_t *parent, const char *what);
int kv_tree_resolve(const mh_kv_batch *b, const int32_t *parent, const char *what);

namespace {

// Lane i's row i of a sequence follows this row of it (as given: loaded ahead
// of what is needed first). Called by whole waves, as the two below.
__device__ __forceinline__ int kv_parent(const int32_t *parent, const KvSeq &q) {
    const int i = threadIdx.x & 63;
    return i < q.n ? parent[q.r0 + i] : -1;
}

// Lane i's row i: itself and the rows before it on its path as bits (none for
// i >= n), p its kv_parent. Paths are joined from their halves: after step o a
// row has the nearest 2^(o + 1) of them, and `p` is the next one.
__device__ __forceinline__ uint64_t kv_paths(int p, const KvSeq &q, unsigned *err) {
    const int i = threadIdx.x & 63;
    if (p < -1 || p >= i) {   // (i >= n: -1)
        if (p != -1) raise_err(err);
        p = -1;
    }
    unsigned long long see = i < q.n ? 1ull << i : 0ull;
    for (int o = 1; o < q.n; o <<= 1) {
        const int from = max(p, 0);
        const unsigned long long s = __shfl(see, from, 64);
        const int pp = __shfl(p, from, 64);
        see |= p >= 0 ? s : 0ull;
        p = p >= 0 ? pp : p;
    }
    return see;
}

// The depth of row `row` of the arrays, a row of sequence q, from the parents
// of the 64 rows that end there (lane i: of row - 63 + i; any value where that
// is no row): they can be on their way before the sequence is known.
__device__ __forceinline__ int kv_depth(int p, const KvSeq &q, int row, unsigned *err) {
    const int lane = threadIdx.x & 63, first = q.r0 - row + 63, i = lane - first;   // first: the lane of the sequence's first row
    if (i < 0) p = -1;
    if (p < -1 || p >= i) {
        if (p != -1) raise_err(err);
        p = -1;
    }
    int d = p >= 0;
    for (int o = 1; o < 64 - first; o <<= 1) {   // (d steps lead from a row to row p, or to the tree's first ones)
        const int from = first + max(p, 0), dd = __shfl(d, from, 64), pp = __shfl(p, from, 64);
        d += p >= 0 ? dd : 0;
        p = p >= 0 ? pp : p;
    }
    return __builtin_amdgcn_readlane(d, 63);
}

// The nearest w rows of a path (a row follows one of a lower number: the
// highest w bits).
__device__ __forceinline__ uint64_t kv_nearest(uint64_t see, int w) {
    for (int n = __popcll(see); n > w; --n) see &= see - 1;
    return see;
}

}  // namespace
}  // namespace mh
