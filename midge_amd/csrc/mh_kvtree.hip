// mh_kvtree.hip — trees of drafted tokens on paged k/v caches: the checks that
// their functions share, and the move of the kept rows (mh_kv_keep_dev).
#include "mh_kvtree.cuh"

#include <algorithm>
#include <vector>

namespace mh {

int kv_tree_validate(const mh_kv_batch *b, const int32_t *parent, const char *what) {
    if (!parent) return fail(MH_E_ARG, "%s: NULL parent", what);
    if ((uintptr_t)parent % 4) return fail(MH_E_ARG, "%s: misaligned parent", what);
    if (b->max_rows > kTreeRows) return fail(MH_E_UNSUPPORTED, "%s: trees of %d rows (at most %d)", what, b->max_rows, kTreeRows);
    return MH_OK;
}

int kv_tree_resolve(const mh_kv_batch *b, const int32_t *parent, const char *what) {
    return resolve_here(parent, 4 * (uint64_t)b->n_rows, what);
}

namespace {

constexpr int kLayers = 64;   // of a launch: their pointers are its arguments (2 KB)

struct KeepArgs {
    KvBatchDev b;
    const int32_t *n_kept, *kept;
    int32_t *len_out;   // NULL: written by another launch
    unsigned *err;
    int64_t n_pages;
    int dt, nkv, hd, shift;
    int heads, parts;   // heads a wave takes, waves for all of them
    uint8_t *mem[kLayers][4];   // k, v, ks, vs
};

// A wave per k or v of a sequence and of some heads (blockIdx.y: layer): lane j
// has row kept[j] and its slots. Rows go down only (kept[j] >= j), so that rows
// read in ascending order, some at a time and all of those before any is
// written, are not written before they are read. Bound by its chain of loads
// (the sequence and its kept rows, their pages, the rows): a wave takes as many
// heads as make a kilobyte of a row.
constexpr int kWaves = 4, kAhead = 8;
__global__ void __launch_bounds__(64 * kWaves) k_kv_keep(KeepArgs A) {
    const int lane = threadIdx.x & 63, w = blockIdx.x * kWaves + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int which = w & 1, layer = blockIdx.y, s = (w >> 1) / A.parts, part = (w >> 1) - s * A.parts;
    if (s >= A.b.n_seqs) return;
    const int from = lane < A.b.max_rows ? A.kept[(int64_t)s * A.b.max_rows + lane] : 0, n = A.n_kept[s];
    KvSeq q;
    if (!kv_tree_seq(A.b, A.shift, s, &q)) {
        raise_err(A.err);
        return;
    }
    const int base = q.len - q.n, before = __shfl_up(from, 1, 64);
    const bool mine = lane < n;
    bool bad = n < 0 || n > q.n || (mine && (from < 0 || from >= q.n || (lane && from <= before)));
    int old_page = 0, new_page = 0;
    if (mine && !bad) {
        const int32_t *pages = A.b.pages + (int64_t)s * A.b.max_pages;
        old_page = pages[(base + from) >> A.shift];
        new_page = pages[(base + lane) >> A.shift];
        bad = from != lane && (old_page < 0 || old_page >= A.n_pages || new_page < 0 || new_page >= A.n_pages);
    }
    if (__ballot(bad)) {
        raise_err(A.err);
        return;
    }
    if (A.len_out && layer == 0 && part == 0 && which == 0 && lane == 0) A.len_out[s] = base + n;
    const unsigned long long moved = __ballot(mine && from != lane);
    if (!moved) return;
    const int first = __builtin_ctzll(moved);   // all from here on
    KvCacheDev c{};
    c.nkv = A.nkv;
    c.shift = A.shift;
    const int in = (1 << A.shift) - 1, h0 = part * A.heads, heads = min(A.heads, A.nkv - h0);
    const unsigned long long src = kv_slot(c, old_page, h0, (base + from) & in), dst = kv_slot(c, new_page, h0, (base + lane) & in);
    auto move = [&](uint8_t *mem, auto unit, unsigned per) {   // `per` units a row of a head
        using T = decltype(unit);
        T *p = (T *)mem;
        const unsigned row = heads * per, all = (n - first) * row;
        for (unsigned u0 = 0; u0 < all; u0 += 64 * kAhead) {
            T v[kAhead];
            unsigned long long to[kAhead];
#pragma unroll
            for (int k = 0; k < kAhead; ++k) {
                const unsigned u = min(u0 + 64 * k + lane, all - 1), j = u / row, r = u - j * row, h = r / per;
                const unsigned long long at = ((unsigned long long)h << A.shift) * per + (r - h * per);
                to[k] = __shfl(dst, first + j, 64) * per + at;
                v[k] = p[__shfl(src, first + j, 64) * per + at];
            }
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");   // all lanes' reads before any write
#pragma unroll
            for (int k = 0; k < kAhead; ++k)
                if (u0 + 64 * k + lane < all) p[to[k]] = v[k];
        }
    };
    const unsigned row = A.dt == MH_KV_F16 ? 2 * A.hd : A.hd / 2;
    move(A.mem[layer][which], mh_u4{}, row / 16);
    if (A.dt != MH_KV_F16) move(A.mem[layer][2 + which], uint8_t{}, A.hd / 32);
}

}  // namespace
}  // namespace mh

using namespace mh;

extern "C" {

int mh_kv_keep_dev(const mh_kv_cache *caches, int n_caches, const mh_kv_batch *b, const int32_t *n_kept, const int32_t *kept,
                   int32_t *len_out) {
    clear_error();
    const char *what = "mh_kv_keep_dev";
    if (!caches || n_caches < 1 || n_caches > 4096) return fail(MH_E_ARG, "%s: %d caches", what, n_caches);
    for (int i = 0; i < n_caches; ++i) {
        const mh_kv_cache &c = caches[i], &f = caches[0];
        MH_TRY(kv_validate(&c, b, what));
        if (c.dt != f.dt || c.n_kv_heads != f.n_kv_heads || c.head_dim != f.head_dim || c.page != f.page || c.n_pages != f.n_pages)
            return fail(MH_E_ARG, "%s: cache %d has another type or shape than the first", what, i);
    }
    if (!n_kept || !kept || !len_out) return fail(MH_E_ARG, "%s: NULL n_kept, kept or len_out", what);
    if (((uintptr_t)n_kept | (uintptr_t)kept | (uintptr_t)len_out) % 4) return fail(MH_E_ARG, "%s: misaligned n_kept, kept or len_out", what);
    if (b->max_rows > kTreeRows) return fail(MH_E_UNSUPPORTED, "%s: trees of %d rows (at most %d)", what, b->max_rows, kTreeRows);
    // what is written apart from everything else: the caches from each other, and all from the arrays
    const bool f16 = caches[0].dt == MH_KV_F16;
    const uint64_t cb = kv_cache_bytes(caches), lb = 4 * (uint64_t)b->n_seqs, kb = lb * b->max_rows;
    struct Range {
        uintptr_t at;
        uint64_t bytes;
        bool written;
    };
    std::vector<Range> mem;
    try {
        mem.reserve(4 * (size_t)n_caches + 6);
    } catch (...) {
        return fail(MH_E_NOMEM, "%s: host memory", what);
    }
    for (int i = 0; i < n_caches; ++i) {
        for (const void *p : {caches[i].k, caches[i].v}) mem.push_back({(uintptr_t)p, cb, true});
        if (!f16)
            for (const void *p : {caches[i].ks, caches[i].vs}) mem.push_back({(uintptr_t)p, cb / 16, true});
    }
    mem.push_back({(uintptr_t)len_out, lb, true});
    mem.push_back({(uintptr_t)n_kept, lb, false});
    mem.push_back({(uintptr_t)kept, kb, false});
    mem.push_back({(uintptr_t)b->len, lb, false});
    mem.push_back({(uintptr_t)b->pages, lb * b->max_pages, false});
    if (b->row0) mem.push_back({(uintptr_t)b->row0, lb + 4, false});
    std::sort(mem.begin(), mem.end(), [](const Range &x, const Range &y) { return x.at < y.at; });
    uintptr_t end = 0, end_written = 0;   // of the ranges so far
    for (const Range &r : mem) {
        if (r.at < (r.written ? end : end_written)) return fail(MH_E_ARG, "%s: memory at %p is named twice", what, (void *)r.at);
        end = std::max<uintptr_t>(end, r.at + r.bytes);
        if (r.written) end_written = std::max<uintptr_t>(end_written, r.at + r.bytes);
    }
    const int nkv = caches[0].n_kv_heads, row = caches[0].head_dim * (f16 ? 4 : 1) / 2, heads = std::min(nkv, std::max(1, 1024 / row)),
              parts = (nkv + heads - 1) / heads;
    const int64_t waves = 2 * (int64_t)b->n_seqs * parts;
    if (waves >= ((int64_t)1 << 25)) return fail(MH_E_UNSUPPORTED, "%s: %d sequences of %d k/v heads", what, b->n_seqs, nkv);
    MH_TRY(require_init());
    OnDevice here;
    KeepArgs A{};
    KvCacheDev cd;
    MH_TRY(kv_resolve(caches, b, &cd, &A.b, what));
    for (int i = 1; i < n_caches; ++i) {
        MH_TRY(resolve_here(caches[i].k, cb, what));
        MH_TRY(resolve_here(caches[i].v, cb, what));
        if (f16) continue;
        MH_TRY(resolve_here(caches[i].ks, cb / 16, what));
        MH_TRY(resolve_here(caches[i].vs, cb / 16, what));
    }
    A.n_pages = cd.n_pages;
    A.dt = cd.dt;
    A.nkv = cd.nkv;
    A.hd = cd.hd;
    A.shift = cd.shift;
    A.heads = heads;
    A.parts = parts;
    MH_TRY(resolve_here(n_kept, lb, what));
    MH_TRY(resolve_here(kept, kb, what));
    MH_TRY(resolve_here(len_out, lb, what));
    MH_TRY(kv_flag(&A.err));
    A.n_kept = n_kept;
    A.kept = kept;
    for (int i = 0; i < n_caches; i += kLayers) {
        const int k = std::min(kLayers, n_caches - i);
        A.len_out = i ? nullptr : len_out;
        for (int j = 0; j < k; ++j) {
            const mh_kv_cache &c = caches[i + j];
            uint8_t *const p[4] = {(uint8_t *)c.k, (uint8_t *)c.v, c.ks, c.vs};
            std::copy(p, p + 4, A.mem[j]);
        }
        MH_LAUNCH("kv_keep", k_kv_keep, dim3((unsigned)((waves + kWaves - 1) / kWaves), (unsigned)k), dim3(64 * kWaves), 0, stream(), A);
    }
    return hip_check(hipGetLastError(), "kv keep launch");
}

}  // extern "C"
