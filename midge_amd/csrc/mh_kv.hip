// mh_kv.hip — paged k/v caches: the argument checks shared by every entry
// point on them, the append of new rows (mh_kv_append_dev) and their
// read-back (mh_kv_read_dev).
//
// The append is attention()'s part between the projections and the scores
// (engine/midge.c:349-368): biases, optional per-head RMSNorm, RoPE, k and v
// into the cache.
#include "mh_kv.cuh"
#include "mh_xchg.cuh"

namespace mh {

int kv_validate(const mh_kv_cache *c, const mh_kv_batch *b, const char *what) {
    if (!c || !b) return fail(MH_E_ARG, "%s: NULL cache or batch", what);
    if (c->dt != MH_KV_F16 && c->dt != MH_KV_MXFP4) return fail(MH_E_DTYPE, "%s: unknown cache type %d", what, c->dt);
    const int hd = c->head_dim, pg = c->page;
    if (hd != 32 && hd != 64 && hd != 96 && hd != 128 && hd != 192 && hd != 256)
        return fail(hd > 0 ? MH_E_UNSUPPORTED : MH_E_ARG, "%s: head_dim %d (32, 64, 96, 128, 192 or 256)", what, hd);
    if (c->n_kv_heads < 1 || c->n_kv_heads > 1024) return fail(MH_E_ARG, "%s: %d k/v heads", what, c->n_kv_heads);
    if (pg < 16 || pg > 4096 || (pg & (pg - 1))) return fail(MH_E_ARG, "%s: pages of %d tokens (a power of two, 16..4096)", what, pg);
    if (c->n_pages < 1 || c->n_pages > INT32_MAX) return fail(MH_E_ARG, "%s: %lld pages", what, (long long)c->n_pages);
    if (!c->k || !c->v || (c->dt == MH_KV_MXFP4 && (!c->ks || !c->vs))) return fail(MH_E_ARG, "%s: NULL cache memory", what);
    if (((uintptr_t)c->k | (uintptr_t)c->v) % 16 || (c->dt == MH_KV_MXFP4 && ((uintptr_t)c->ks | (uintptr_t)c->vs) % 16))
        return fail(MH_E_ARG, "%s: cache memory is not 16-byte aligned", what);
    if (b->n_seqs < 1 || b->n_seqs > (1 << 20) || b->n_rows < 0 || b->n_rows > (1 << 24))
        return fail(MH_E_ARG, "%s: %d sequences, %d rows", what, b->n_seqs, b->n_rows);
    if (b->max_rows < 1) return fail(MH_E_ARG, "%s: max_rows %d", what, b->max_rows);
    if (b->max_pages < 1 || (int64_t)b->max_pages * pg > INT32_MAX - 4096)
        return fail(MH_E_ARG, "%s: %d pages of %d tokens a sequence", what, b->max_pages, pg);
    if (!b->len || !b->pages) return fail(MH_E_ARG, "%s: NULL len or pages", what);
    if (!b->row0 && b->n_rows != b->n_seqs)
        return fail(MH_E_ARG, "%s: without row0 a sequence has one row (%d rows, %d sequences)", what, b->n_rows, b->n_seqs);
    if (((uintptr_t)b->row0 | (uintptr_t)b->len | (uintptr_t)b->pages) % 4) return fail(MH_E_ARG, "%s: misaligned row0, len or pages", what);
    return MH_OK;
}

int kv_resolve(const mh_kv_cache *c, const mh_kv_batch *b, KvCacheDev *cd, KvBatchDev *bd, const char *what) {
    const uint64_t n = (uint64_t)c->n_pages * c->n_kv_heads * c->page * c->head_dim;
    const uint64_t bytes = c->dt == MH_KV_F16 ? 2 * n : n / 2;
    MH_TRY(resolve_here(c->k, bytes, what));
    MH_TRY(resolve_here(c->v, bytes, what));
    if (c->dt == MH_KV_MXFP4) {
        MH_TRY(resolve_here(c->ks, n / 32, what));
        MH_TRY(resolve_here(c->vs, n / 32, what));
    }
    if (b->row0) MH_TRY(resolve_here(b->row0, 4 * ((uint64_t)b->n_seqs + 1), what));
    MH_TRY(resolve_here(b->len, 4 * (uint64_t)b->n_seqs, what));
    MH_TRY(resolve_here(b->pages, 4 * (uint64_t)b->n_seqs * b->max_pages, what));
    *cd = KvCacheDev{(uint8_t *)c->k, (uint8_t *)c->v, c->ks, c->vs, c->n_pages, c->dt, c->n_kv_heads, c->head_dim,
                     __builtin_ctz((unsigned)c->page)};
    *bd = KvBatchDev{b->row0, b->len, b->pages, b->n_seqs, b->n_rows, b->max_rows, b->max_pages};
    return MH_OK;
}

namespace {

constexpr int kWaves = 4;

// f32 -> f16 as wk_to_f16 (engine/mkern.h:261-273): nearest even, magnitudes
// below the normal range to a signed zero.
__device__ __forceinline__ uint16_t kv_f16(float f) {
    const _Float16 h = (_Float16)f;
    uint16_t u;
    __builtin_memcpy(&u, &h, 2);
    const uint32_t b = __float_as_uint(f);
    return ((b >> 23) & 0xffu) < 113u ? (uint16_t)((b >> 16) & 0x8000u) : u;
}

// The sequence that has row `row` and its place there; false for a row of no
// sequence (or of one out of bounds, which raises the error).
__device__ __forceinline__ bool find_row(const KvBatchDev &b, int shift, int row, int *seq, KvSeq *q, unsigned *err) {
    int s = row;
    if (b.row0) {   // the number of ends at or before the row
        int lo = 0, hi = b.n_seqs;
        while (lo < hi) {
            const int m = (lo + hi) >> 1;
            if (b.row0[m + 1] <= row) lo = m + 1;
            else hi = m;
        }
        s = lo;
    }
    if (s >= b.n_seqs) return false;
    *seq = s;
    if (!kv_seq(b, shift, s, q)) {
        raise_err(err);
        return false;
    }
    return row >= q->r0 && row < q->r0 + q->n;
}

struct AppendArgs {
    KvCacheDev c;
    KvBatchDev b;
    const float *q, *k, *v, *bq, *bk, *bv, *qn, *kn, *co, *si;
    float *q_out;
    int64_t ldq, ldk, ldv;
    unsigned *err;
    int nh, ctx;
    float eps;
};

// One wave per head of a row (nh of q, nkv of k, nkv of v), lanes over its
// elements.
__global__ void __launch_bounds__(64 * kWaves) k_kv_append(AppendArgs A) {
    __shared__ double u[kWaves][256];
    __shared__ float f[kWaves][256];
    const int wv = threadIdx.x >> 6, lane = threadIdx.x & 63, hd = A.c.hd, half = hd / 2;
    const int per = A.nh + 2 * A.c.nkv;
    const int64_t unit = (int64_t)blockIdx.x * kWaves + wv;
    const int row = (int)(unit / per), hu = (int)(unit % per);
    const int kind = hu < A.nh ? 0 : hu < A.nh + A.c.nkv ? 1 : 2, head = kind == 0 ? hu : kind == 1 ? hu - A.nh : hu - A.nh - A.c.nkv;
    int seq = 0, pos = -1, page = -1;
    KvSeq sq{};
    bool live = row < A.b.n_rows && find_row(A.b, A.c.shift, row, &seq, &sq, A.err);
    if (live) pos = sq.len - sq.n + (row - sq.r0);
    live = live && pos >= 0;
    if (live && A.co && pos >= A.ctx) {
        raise_err(A.err);
        live = false;
    }
    if (live && kind) {
        page = A.b.pages[(int64_t)seq * A.b.max_pages + (pos >> A.c.shift)];
        if (!kv_page_ok(A.c, page)) {
            raise_err(A.err);
            live = false;
        }
    }
    const float *x = kind == 0 ? A.q + (int64_t)row * A.ldq : kind == 1 ? A.k + (int64_t)row * A.ldk : A.v + (int64_t)row * A.ldv;
    const float *bias = kind == 0 ? A.bq : kind == 1 ? A.bk : A.bv, *norm = kind == 0 ? A.qn : kind == 1 ? A.kn : nullptr;
    double ss = 0.0;
    if (live)
        for (int e = lane; e < hd; e += 64) {
            double t = x[head * hd + e];
            if (bias) t += (double)bias[head * hd + e];
            u[wv][e] = t;
            ss += t * t;
        }
    if (live && norm) {
        for (int o = 32; o; o >>= 1) ss += __shfl_xor(ss, o, 64);
        const double inv = 1.0 / sqrt(ss / hd + (double)A.eps);
        for (int e = lane; e < hd; e += 64) u[wv][e] = u[wv][e] * inv * (double)norm[e];
    }
    __syncthreads();
    if (live)
        for (int e = lane; e < hd; e += 64) {
            double t = u[wv][e];
            if (A.co && kind < 2) {
                const int i = e < half ? e : e - half;
                const double cs = A.co[(int64_t)pos * half + i], sn = A.si[(int64_t)pos * half + i];
                t = e < half ? t * cs - u[wv][e + half] * sn : t * cs + u[wv][e - half] * sn;
            }
            f[wv][e] = (float)t;
        }
    __syncthreads();
    if (!live) return;
    if (kind == 0) {
        for (int e = lane; e < hd; e += 64) A.q_out[((int64_t)row * A.nh + head) * hd + e] = f[wv][e];
        return;
    }
    const uint64_t slot = kv_slot(A.c, page, head, pos & ((1 << A.c.shift) - 1));
    uint8_t *dst = kind == 1 ? A.c.k : A.c.v, *exps = kind == 1 ? A.c.ks : A.c.vs;
    if (A.c.dt == MH_KV_F16) {
        uint16_t *d16 = (uint16_t *)dst + slot * hd;
        for (int e = lane; e < hd; e += 64) d16[e] = kv_f16(f[wv][e]);
        return;
    }
    for (int b = lane; b < hd / 2; b += 64) {   // bytes of two codes
        const int blk = b / 16;
        uint32_t top = 0;
        for (int j = 0; j < 32; ++j) top = max(top, __float_as_uint(f[wv][32 * blk + j]) & 0x7fffffffu);
        const int eb = kv_block_exp(top);
        const float inv = eb == 255 ? 0.f : kv_scale((uint32_t)(254 - eb));
        dst[slot * (hd / 2) + b] = (uint8_t)(kv_code(f[wv][2 * b], inv) | kv_code(f[wv][2 * b + 1], inv) << 4);
        if (b % 16 == 0) exps[slot * (hd / 32) + blk] = (uint8_t)eb;
    }
}

// The stored values of a row, one wave per k/v head (k then v).
__global__ void __launch_bounds__(64 * kWaves) k_kv_read(KvCacheDev c, KvBatchDev b, float *ko, float *vo, unsigned *err) {
    const int wv = threadIdx.x >> 6, lane = threadIdx.x & 63, hd = c.hd;
    const int64_t unit = (int64_t)blockIdx.x * kWaves + wv;
    const int row = (int)(unit / (2 * c.nkv)), hu = (int)(unit % (2 * c.nkv)), head = hu % c.nkv;
    float *out = hu < c.nkv ? ko : vo;
    int seq;
    KvSeq q;
    if (!out || row >= b.n_rows || !find_row(b, c.shift, row, &seq, &q, err)) return;
    const int pos = q.len - q.n + (row - q.r0);
    if (pos < 0) return;
    const int page = b.pages[(int64_t)seq * b.max_pages + (pos >> c.shift)];
    if (!kv_page_ok(c, page)) {
        if (lane == 0) raise_err(err);
        return;
    }
    const uint64_t slot = kv_slot(c, page, head, pos & ((1 << c.shift) - 1));
    const uint8_t *src = hu < c.nkv ? c.k : c.v, *exps = hu < c.nkv ? c.ks : c.vs;
    out += ((int64_t)row * c.nkv + head) * hd;
    for (int e = lane; e < hd; e += 64) {
        if (c.dt == MH_KV_F16) {
            out[e] = mh_f16(((const uint16_t *)src)[slot * hd + e]);
        } else {
            const uint32_t w = src[slot * (hd / 2) + e / 2];
            const mh_v2f p = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.0f, 0);
            out[e] = (e & 1 ? p.y : p.x) * kv_scale(exps[slot * (hd / 32) + e / 32]);
        }
    }
}

}  // namespace
}  // namespace mh

using namespace mh;

extern "C" {

int mh_kv_append_dev(const mh_kv_cache *c, const mh_kv_batch *b, const mh_kv_rows *r) {
    clear_error();
    const char *what = "mh_kv_append_dev";
    MH_TRY(kv_validate(c, b, what));
    if (!r || !r->q || !r->k || !r->v || !r->q_out) return fail(MH_E_ARG, "%s: NULL rows", what);
    const int hd = c->head_dim, nh = r->n_heads, nkv = c->n_kv_heads;
    if (nh < 1 || nh > 65536 || nh % nkv) return fail(MH_E_ARG, "%s: %d query heads on %d k/v heads", what, nh, nkv);
    const int64_t qd = (int64_t)nh * hd, kvd = (int64_t)nkv * hd;
    const int64_t far = (int64_t)1 << 40;
    if (r->ldq < qd || r->ldk < kvd || r->ldv < kvd || r->ldq > far || r->ldk > far || r->ldv > far)
        return fail(MH_E_ARG, "%s: rows of %lld, %lld, %lld floats do not hold the heads", what, (long long)r->ldq, (long long)r->ldk,
                    (long long)r->ldv);
    if (!r->rope_cos != !r->rope_sin) return fail(MH_E_ARG, "%s: one rotation table without the other", what);
    if (r->rope_cos && r->ctx < 1) return fail(MH_E_ARG, "%s: rotation tables of %d positions", what, r->ctx);
    if (!(r->norm_eps >= 0.f) && (r->qn || r->kn)) return fail(MH_E_ARG, "%s: norm_eps %g", what, (double)r->norm_eps);
    if (((uintptr_t)r->q | (uintptr_t)r->k | (uintptr_t)r->v | (uintptr_t)r->q_out) % 4) return fail(MH_E_ARG, "%s: misaligned rows", what);
    if (b->n_rows) {
        const uint64_t last = (uint64_t)b->n_rows - 1, qb = 4 * (last * r->ldq + qd), kb = 4 * (last * r->ldk + kvd),
                       vb = 4 * (last * r->ldv + kvd), ob = 4 * (uint64_t)b->n_rows * qd;
        if (!(r->q_out == r->q && r->ldq == qd) && kv_overlap(r->q_out, ob, r->q, qb))
            return fail(MH_E_ARG, "%s: q_out overlaps q (it may be q itself where ldq is the heads' width)", what);
        if (kv_overlap(r->q_out, ob, r->k, kb) || kv_overlap(r->q_out, ob, r->v, vb)) return fail(MH_E_ARG, "%s: q_out overlaps k or v", what);
    }
    MH_TRY(require_init());
    if (!b->n_rows) return MH_OK;
    OnDevice here;
    AppendArgs A{};
    MH_TRY(kv_resolve(c, b, &A.c, &A.b, what));
    const uint64_t last = (uint64_t)b->n_rows - 1;
    MH_TRY(resolve_here(r->q, 4 * (last * r->ldq + qd), what));
    MH_TRY(resolve_here(r->k, 4 * (last * r->ldk + kvd), what));
    MH_TRY(resolve_here(r->v, 4 * (last * r->ldv + kvd), what));
    MH_TRY(resolve_here(r->q_out, 4 * (uint64_t)b->n_rows * qd, what));
    const struct {
        const float *p;
        uint64_t n;
        const float **to;
    } w[] = {{r->bq, (uint64_t)qd, &A.bq}, {r->bk, (uint64_t)kvd, &A.bk}, {r->bv, (uint64_t)kvd, &A.bv},
             {r->qn, (uint64_t)hd, &A.qn}, {r->kn, (uint64_t)hd, &A.kn},
             {r->rope_cos, (uint64_t)r->ctx * (hd / 2), &A.co}, {r->rope_sin, (uint64_t)r->ctx * (hd / 2), &A.si}};
    for (const auto &t : w)
        if (t.p) {
            const void *d;
            MH_TRY(resolve_weight(t.p, 4 * t.n, &d, what));
            *t.to = (const float *)d;
        }
    A.q = r->q;
    A.k = r->k;
    A.v = r->v;
    A.q_out = r->q_out;
    A.ldq = r->ldq;
    A.ldk = r->ldk;
    A.ldv = r->ldv;
    A.nh = nh;
    A.ctx = r->ctx;
    A.eps = r->norm_eps;
    MH_TRY(kv_flag(&A.err));
    const int64_t units = (int64_t)b->n_rows * (nh + 2 * nkv), blocks = (units + kWaves - 1) / kWaves;
    if (blocks > INT32_MAX) return fail(MH_E_UNSUPPORTED, "%s: %lld head rows in one call", what, (long long)units);
    MH_LAUNCH("kv_append", k_kv_append, dim3((unsigned)blocks), dim3(64 * kWaves), 0, stream(), A);
    return hip_check(hipGetLastError(), "kv append launch");
}

int mh_kv_read_dev(const mh_kv_cache *c, const mh_kv_batch *b, float *k, float *v) {
    clear_error();
    const char *what = "mh_kv_read_dev";
    MH_TRY(kv_validate(c, b, what));
    if (!k && !v) return fail(MH_E_ARG, "%s: neither k nor v wanted", what);
    if (((uintptr_t)k | (uintptr_t)v) % 4) return fail(MH_E_ARG, "%s: misaligned output", what);
    const uint64_t bytes = 4 * (uint64_t)b->n_rows * c->n_kv_heads * c->head_dim;
    if (k && v && kv_overlap(k, bytes, v, bytes)) return fail(MH_E_ARG, "%s: k overlaps v", what);
    MH_TRY(require_init());
    if (!b->n_rows) return MH_OK;
    OnDevice here;
    KvCacheDev cd;
    KvBatchDev bd;
    MH_TRY(kv_resolve(c, b, &cd, &bd, what));
    if (k) MH_TRY(resolve_here(k, bytes, what));
    if (v) MH_TRY(resolve_here(v, bytes, what));
    unsigned *err;
    MH_TRY(kv_flag(&err));
    const int64_t units = (int64_t)b->n_rows * 2 * c->n_kv_heads, blocks = (units + kWaves - 1) / kWaves;
    if (blocks > INT32_MAX) return fail(MH_E_UNSUPPORTED, "%s: %lld head rows in one call", what, (long long)units);
    MH_LAUNCH("kv_read", k_kv_read, dim3((unsigned)blocks), dim3(64 * kWaves), 0, stream(), cd, bd, k, v, err);
    return hip_check(hipGetLastError(), "kv read launch");
}

int mh_kv_check(const mh_kv_cache *c, const mh_kv_batch *b) {
    clear_error();
    MH_TRY(kv_validate(c, b, "mh_kv_check"));
    KvCacheDev cd{};
    cd.n_pages = c->n_pages;
    const int shift = __builtin_ctz((unsigned)c->page);
    const KvBatchDev bd{b->row0, b->len, b->pages, b->n_seqs, b->n_rows, b->max_rows, b->max_pages};
    for (int s = 0; s < b->n_seqs; ++s) {
        KvSeq q;
        if (!kv_seq(bd, shift, s, &q))
            return fail(MH_E_RANGE, "mh_kv_check: sequence %d: rows %d + %d of %d (at most %d), %d tokens on %d pages", s, q.r0, q.n,
                        b->n_rows, b->max_rows, q.len, b->max_pages);
        for (int64_t t = 0; t < q.len; t += c->page) {
            const int p = b->pages[(int64_t)s * b->max_pages + (t >> shift)];
            if (!kv_page_ok(cd, p))
                return fail(MH_E_RANGE, "mh_kv_check: sequence %d: page %d of %lld holds token %lld", s, p, (long long)c->n_pages, (long long)t);
        }
    }
    return MH_OK;
}

}  // extern "C"
