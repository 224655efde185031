// mh_kvattn.hip — attention of a batch's rows over a paged k/v cache
// (mh_kv_attention_dev): attention()'s scores, softmax and weighted sum
// (engine/midge.c:371-396) for many sequences, from f16 or MXFP4.
#include <math.h>

#include "mh_kv.cuh"
#include "mh_xchg.cuh"

namespace mh {
namespace {

struct KvAttnArgs {
    KvCacheDev c;
    KvBatchDev b;
    const float *q, *sink;
    float *out;
    unsigned *err;
    int nh, group, window;
    float scale;
};

__device__ __forceinline__ float kv_value(const KvCacheDev &c, const uint8_t *src, const uint8_t *exps, uint64_t slot, int e) {
    if (c.dt == MH_KV_F16) return mh_f16(((const uint16_t *)src)[slot * c.hd + e]);
    const uint32_t w = src[slot * (c.hd / 2) + e / 2];
    const mh_v2f p = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.0f, 0);
    return (e & 1 ? p.y : p.x) * kv_scale(exps[slot * (c.hd / 32) + e / 32]);
}

// Block (sequence's row i, head h): 256 tokens at a time, a thread a token
// for the scores, then a thread a dim for the weighted sum.
__global__ void __launch_bounds__(256) k_kv_attn_rows(KvAttnArgs A) {
    __shared__ float qs[256], sc[256], red[4];
    __shared__ uint64_t sl[256];
    const int s = blockIdx.z, i = blockIdx.x, h = blockIdx.y, kh = h / A.group, t = threadIdx.x, hd = A.c.hd;
    KvSeq q;
    if (!kv_seq(A.b, A.c.shift, s, &q)) {
        if (t == 0) raise_err(A.err);
        return;
    }
    if (i >= q.n) return;
    const int64_t o = ((int64_t)(q.r0 + i) * A.nh + h) * hd;
    const int pos = q.len - q.n + i, lo = A.window > 0 ? max(0, pos + 1 - A.window) : 0;
    if (t < hd) qs[t] = A.q[o + t];
    __syncthreads();
    float m = -INFINITY, l = 0.f, acc = 0.f;
    for (int base = lo; base <= pos; base += 256) {
        const int n = min(256, pos + 1 - base);
        float x = -INFINITY;
        if (t < n) {
            const int tok = base + t, page = A.b.pages[(int64_t)s * A.b.max_pages + (tok >> A.c.shift)];
            const bool ok = kv_page_ok(A.c, page);
            if (!ok) raise_err(A.err);
            const uint64_t slot = kv_slot(A.c, ok ? page : 0, kh, tok & ((1 << A.c.shift) - 1));
            sl[t] = slot;
            float d = 0.f;
            for (int e = 0; e < hd; ++e) d = fmaf(qs[e], kv_value(A.c, A.c.k, A.c.ks, slot, e), d);
            x = ok ? d * A.scale : NAN;
        }
        float mx = x;
        for (int j = 32; j; j >>= 1) mx = fmaxf(mx, __shfl_xor(mx, j, 64));
        if ((t & 63) == 0) red[t >> 6] = mx;
        __syncthreads();
        const float mn = fmaxf(m, fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3])));
        const float p = t < n ? expf(x - mn) : 0.f, al = m == mn ? 1.f : expf(m - mn);
        float ps = p;
        for (int j = 32; j; j >>= 1) ps += __shfl_xor(ps, j, 64);
        sc[t] = p;
        __syncthreads();
        if ((t & 63) == 0) red[t >> 6] = ps;
        __syncthreads();
        l = l * al + (red[0] + red[1] + red[2] + red[3]);
        m = mn;
        if (t < hd) {
            acc *= al;
            for (int j = 0; j < n; ++j) acc = fmaf(sc[j], kv_value(A.c, A.c.v, A.c.vs, sl[j], t), acc);
        }
        __syncthreads();
    }
    if (A.sink) {
        const float sk = A.sink[h], mn = fmaxf(m, sk), al = m == mn ? 1.f : expf(m - mn);
        acc *= al;
        l = l * al + (sk == mn ? 1.f : expf(sk - mn));
    }
    if (t < hd) A.out[o + t] = pos < 0 ? 0.f : acc / l;
}

}  // namespace
}  // namespace mh

using namespace mh;

extern "C" {

int mh_kv_attention_ws(const mh_kv_cache *c, const mh_kv_batch *b, int n_heads, uint64_t *bytes) {
    clear_error();
    MH_TRY(kv_validate(c, b, "mh_kv_attention_ws"));
    if (!bytes) return fail(MH_E_ARG, "mh_kv_attention_ws: NULL result");
    if (n_heads < 1 || n_heads > 65535 || n_heads % c->n_kv_heads)
        return fail(MH_E_ARG, "mh_kv_attention_ws: %d query heads on %d k/v heads", n_heads, c->n_kv_heads);
    *bytes = 16;
    return MH_OK;
}

int mh_kv_attention_dev(const mh_kv_cache *c, const mh_kv_batch *b, int n_heads, int window, float scale, const float *sink,
                        const float *q, float *out, void *ws, uint64_t ws_bytes) {
    const char *what = "mh_kv_attention_dev";
    uint64_t need = 0;
    MH_TRY(mh_kv_attention_ws(c, b, n_heads, &need));
    if (!q || !out || !ws) return fail(MH_E_ARG, "%s: NULL q, out or workspace", what);
    if (window < 0) return fail(MH_E_ARG, "%s: window %d", what, window);
    if (!std::isfinite(scale)) return fail(MH_E_ARG, "%s: scale %g", what, (double)scale);
    if (ws_bytes < need) return fail(MH_E_ARG, "%s: a workspace of %llu bytes, %llu needed", what, (unsigned long long)ws_bytes,
                                     (unsigned long long)need);
    if (((uintptr_t)q | (uintptr_t)out) % 4 || (uintptr_t)ws % 16) return fail(MH_E_ARG, "%s: misaligned q, out or workspace", what);
    const uint64_t bytes = 4 * (uint64_t)b->n_rows * n_heads * c->head_dim;
    if (kv_overlap(q, bytes, out, bytes)) return fail(MH_E_ARG, "%s: out overlaps q", what);
    MH_TRY(require_init());
    if (!b->n_rows) return MH_OK;
    OnDevice here;
    KvAttnArgs A{};
    MH_TRY(kv_resolve(c, b, &A.c, &A.b, what));
    MH_TRY(resolve_here(q, bytes, what));
    MH_TRY(resolve_here(out, bytes, what));
    MH_TRY(resolve_here(ws, need, what));
    if (sink) {
        const void *d;
        MH_TRY(resolve_weight(sink, 4 * (uint64_t)n_heads, &d, what));
        A.sink = (const float *)d;
    }
    MH_TRY(kv_flag(&A.err));
    A.q = q;
    A.out = out;
    A.nh = n_heads;
    A.group = n_heads / c->n_kv_heads;
    A.window = window;
    A.scale = scale;
    const int mr = b->row0 ? std::min(b->max_rows, b->n_rows) : 1;
    for (int s0 = 0; s0 < b->n_seqs; s0 += 65535) {
        KvAttnArgs P = A;
        P.b.row0 = A.b.row0 ? A.b.row0 + s0 : nullptr;
        P.b.len += s0;
        P.b.pages += (int64_t)s0 * A.b.max_pages;
        MH_LAUNCH("kv_attn", k_kv_attn_rows, dim3((unsigned)mr, (unsigned)n_heads, (unsigned)std::min(65535, b->n_seqs - s0)), dim3(256),
                  0, stream(), P);
    }
    return hip_check(hipGetLastError(), "kv attention launch");
}

}  // extern "C"
