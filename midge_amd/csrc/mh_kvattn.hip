// mh_kvattn.hip — attention of a batch's rows over a paged k/v cache
// (mh_kv_attention_dev, mh_kv_tree_attention_dev): attention()'s scores,
// softmax and weighted sum (engine/midge.c:371-396) for many sequences, from
// f16 or MXFP4.
#include "mh_kvfew.cuh"

namespace mh {

uint64_t kv_few_ws(const mh_kv_cache &c, const mh_kv_batch &b, int group) { return few_ws(c, b, kv_columns(b, group)); }

int kv_few_run(const mh_kv_cache &c, const mh_kv_batch &b, KvAttnArgs A, void *ws) { return few_run<false>(c, b, A, ws); }

int kv_attention_ws(const mh_kv_cache *c, const mh_kv_batch *b, bool tree, int n_heads, uint64_t *bytes, const char *what) {
    clear_error();
    MH_TRY(kv_validate(c, b, what));
    if (!bytes) return fail(MH_E_ARG, "%s: NULL result", what);
    if (n_heads < 1 || n_heads > 65535 || n_heads % c->n_kv_heads)
        return fail(MH_E_ARG, "%s: %d query heads on %d k/v heads", what, n_heads, c->n_kv_heads);
    const int group = n_heads / c->n_kv_heads;
    *bytes = kv_is_few(*c, *b, group, tree) ? kv_few_ws(*c, *b, group) : kv_many_ws(*c, *b, group);
    return MH_OK;
}

// Checks, resolution and launch of both entry points.
static int attention(const mh_kv_cache *c, const mh_kv_batch *b, bool tree, const int32_t *parent, int n_heads, int window, float scale,
                     const float *sink, const float *q, float *out, void *ws, uint64_t ws_bytes, const char *what) {
    uint64_t need = 0;
    MH_TRY(kv_attention_ws(c, b, tree, n_heads, &need, what));
    if (tree) MH_TRY(kv_tree_validate(b, parent, what));
    if (!q || !out || !ws) return fail(MH_E_ARG, "%s: NULL q, out or workspace", what);
    if (window < 0) return fail(MH_E_ARG, "%s: window %d", what, window);
    const float qscale = scale * 1.44269504088896341f;
    if (!std::isfinite(qscale)) return fail(MH_E_ARG, "%s: scale %g", what, (double)scale);
    if (ws_bytes < need) return fail(MH_E_ARG, "%s: a workspace of %llu bytes, %llu needed", what, (unsigned long long)ws_bytes,
                                     (unsigned long long)need);
    if (((uintptr_t)q | (uintptr_t)out | (uintptr_t)ws) % 16) return fail(MH_E_ARG, "%s: misaligned q, out or workspace", what);
    if ((uintptr_t)sink % 4) return fail(MH_E_ARG, "%s: misaligned sinks", what);
    const uint64_t bytes = 4 * (uint64_t)b->n_rows * n_heads * c->head_dim;
    if (kv_overlap(q, bytes, out, bytes)) return fail(MH_E_ARG, "%s: out overlaps q", what);
    if (kv_overlap(ws, need, q, bytes) || kv_overlap(ws, need, out, bytes)) return fail(MH_E_ARG, "%s: the workspace overlaps q or out", what);
    if (tree && (kv_overlap(parent, 4 * (uint64_t)b->n_rows, out, bytes) || kv_overlap(parent, 4 * (uint64_t)b->n_rows, ws, need)))
        return fail(MH_E_ARG, "%s: out or the workspace overlaps parent", what);
    const uint64_t sb = 4 * (uint64_t)n_heads;
    auto sink_apart = [&](const void *p) { return !kv_overlap(p, sb, out, bytes) && !kv_overlap(p, sb, ws, need); };
    if (sink && !sink_apart(sink)) return fail(MH_E_ARG, "%s: out or the workspace overlaps the sinks", what);
    // (grids of 2^32 threads, and quotients of unit numbers as doubles: kv_div)
    if ((int64_t)b->n_seqs * c->n_kv_heads >= (1 << 24) ||
        (double)std::min(b->n_seqs, 256) * ((double)b->max_pages * c->page / 32 + 8) > 0x1p31 ||   // (block_scan)
        ((double)b->n_seqs + (double)b->n_rows * n_heads / c->n_kv_heads / 128) * c->n_kv_heads * ((double)b->max_pages * c->page / 32 + 8) > 0x1p41)
        return fail(MH_E_UNSUPPORTED, "%s: %d sequences of %d k/v heads", what, b->n_seqs, c->n_kv_heads);
    MH_TRY(require_init());
    if (!b->n_rows) return MH_OK;
    OnDevice here;
    KvAttnArgs A{};
    MH_TRY(kv_resolve(c, b, &A.c, &A.b, what));
    if (tree) MH_TRY(kv_tree_resolve(b, parent, what));
    MH_TRY(resolve_here(q, bytes, what));
    MH_TRY(resolve_here(out, bytes, what));
    MH_TRY(resolve_here(ws, need, what));
    MH_TRY(kv_apart(c, b, out, bytes, what));
    MH_TRY(kv_apart(c, b, ws, need, what));
    if (sink) {
        const void *d;
        MH_TRY(resolve_weight(sink, sb, &d, what, true));
        if (!sink_apart(d)) return fail(MH_E_ARG, "%s: out or the workspace overlaps the sinks", what);
        A.sink = (const float *)d;
    }
    MH_TRY(kv_flag(&A.err));
    A.q = q;
    A.out = out;
    A.nh = n_heads;
    A.group = n_heads / c->n_kv_heads;
    A.window = (int64_t)window < (int64_t)b->max_pages * c->page ? window : 0;   // (no length reaches it)
    A.qscale = qscale;
    A.parent = parent;
    if (kv_is_few(*c, *b, A.group, tree)) return tree ? kv_few_tree_run(*c, *b, A, ws) : kv_few_run(*c, *b, A, ws);
    return tree ? kv_many_tree_run(*c, *b, A, ws) : kv_many_run(*c, *b, A, ws);
}

}  // namespace mh

using namespace mh;

extern "C" {

int mh_kv_attention_ws(const mh_kv_cache *c, const mh_kv_batch *b, int n_heads, uint64_t *bytes) {
    return kv_attention_ws(c, b, false, n_heads, bytes, "mh_kv_attention_ws");
}

int mh_kv_attention_dev(const mh_kv_cache *c, const mh_kv_batch *b, int n_heads, int window, float scale, const float *sink,
                        const float *q, float *out, void *ws, uint64_t ws_bytes) {
    return attention(c, b, false, nullptr, n_heads, window, scale, sink, q, out, ws, ws_bytes, "mh_kv_attention_dev");
}

int mh_kv_tree_attention_ws(const mh_kv_cache *c, const mh_kv_batch *b, int n_heads, uint64_t *bytes) {
    MH_TRY(kv_attention_ws(c, b, true, n_heads, bytes, "mh_kv_tree_attention_ws"));
    if (b->max_rows > kTreeRows) return fail(MH_E_UNSUPPORTED, "mh_kv_tree_attention_ws: trees of %d rows (at most %d)", b->max_rows, kTreeRows);
    return MH_OK;
}

int mh_kv_tree_attention_dev(const mh_kv_cache *c, const mh_kv_batch *b, const int32_t *parent, int n_heads, int window, float scale,
                             const float *sink, const float *q, float *out, void *ws, uint64_t ws_bytes) {
    return attention(c, b, true, parent, n_heads, window, scale, sink, q, out, ws, ws_bytes, "mh_kv_tree_attention_dev");
}

}  // extern "C"
