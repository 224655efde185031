// mh_kv.hip — paged k/v caches: the argument checks shared by every entry
// point on them, the append of new rows (mh_kv_append_dev; of trees:
// mh_kv_tree_append_dev) and their read-back (mh_kv_read_dev).
//
// The append is attention()'s part between the projections and the scores
// (engine/midge.c:349-368): biases, optional per-head RMSNorm, RoPE, k and v
// into the cache.
#include "mh_kvtree.cuh"

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
    if (b->n_seqs < 1 || b->n_seqs > (1 << 20) || b->n_rows < 0 || b->n_rows >= (1 << 24))   // (grids of 2^32 threads)
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

uint64_t kv_cache_bytes(const mh_kv_cache *c) {
    const uint64_t n = (uint64_t)c->n_pages * c->n_kv_heads * c->page * c->head_dim;
    return c->dt == MH_KV_F16 ? 2 * n : n / 2;
}

static int apart_from_cache(const mh_kv_cache *c, const void *p, uint64_t bytes, const char *what) {
    const uint64_t n = kv_cache_bytes(c), ne = c->dt == MH_KV_F16 ? 0 : n / 16;
    if (kv_overlap(p, bytes, c->k, n) || kv_overlap(p, bytes, c->v, n) || (ne && (kv_overlap(p, bytes, c->ks, ne) || kv_overlap(p, bytes, c->vs, ne))))
        return fail(MH_E_ARG, "%s: %p overlaps the cache", what, p);
    return MH_OK;
}

int kv_apart(const mh_kv_cache *c, const mh_kv_batch *b, const void *p, uint64_t bytes, const char *what) {
    MH_TRY(apart_from_cache(c, p, bytes, what));
    if ((b->row0 && kv_overlap(p, bytes, b->row0, 4 * ((uint64_t)b->n_seqs + 1))) || kv_overlap(p, bytes, b->len, 4 * (uint64_t)b->n_seqs) ||
        kv_overlap(p, bytes, b->pages, 4 * (uint64_t)b->n_seqs * b->max_pages))
        return fail(MH_E_ARG, "%s: %p overlaps row0, len or pages", what, p);
    return MH_OK;
}

int kv_resolve(const mh_kv_cache *c, const mh_kv_batch *b, KvCacheDev *cd, KvBatchDev *bd, const char *what) {
    const uint64_t bytes = kv_cache_bytes(c);
    MH_TRY(resolve_here(c->k, bytes, what));
    MH_TRY(resolve_here(c->v, bytes, what));
    if (c->dt == MH_KV_MXFP4) {
        MH_TRY(resolve_here(c->ks, bytes / 16, what));
        MH_TRY(resolve_here(c->vs, bytes / 16, what));
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
// below the normal range to a signed zero. (A NaN stays one.)
__device__ __forceinline__ uint16_t kv_f16(float f) {
    const _Float16 h = (_Float16)f;
    uint16_t u;
    __builtin_memcpy(&u, &h, 2);
    const uint32_t b = __float_as_uint(f);
    return ((b >> 23) & 0xffu) < 113u ? (uint16_t)((b >> 16) & 0x8000u) : u;
}

// The sequence that has row `row` and its place there; false for a row of no
// sequence (or of one out of bounds, which raises the error). The row is the
// same for the wave: 64 ends are looked at together.
template <bool TREE>
__device__ __forceinline__ bool find_row(const KvBatchDev &b, int shift, int row, int *seq, KvSeq *q, unsigned *err) {
    int s = row;
    if (b.row0) {   // the number of ends at or before the row, in [lo, hi]
        int lo = 0, hi = b.n_seqs;
        while (lo < hi) {
            const int step = (hi - lo + 63) / 64, i = lo + (int)(threadIdx.x & 63) * step;
            const int n = __popcll(__ballot(i < hi && b.row0[i + 1] <= row));
            hi = min(hi, lo + n * step);
            lo = n ? lo + (n - 1) * step + 1 : lo;
        }
        s = lo;
    }
    if (s >= b.n_seqs) return false;
    *seq = s;
    if (!kv_rows_of<TREE>(b, shift, s, q)) {
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
    const int32_t *parent;   // trees: of each row
};

// Four floats at p: one 16-byte access where the address allows.
__device__ __forceinline__ void load4(const float *p, float *v) {
    if ((uintptr_t)p % 16 == 0) {
        const float4 a = *(const float4 *)p;
        v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w;
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = p[i];
    }
}
__device__ __forceinline__ void store4(float *p, const float *v) {
    if ((uintptr_t)p % 16 == 0) {
        *(float4 *)p = make_float4(v[0], v[1], v[2], v[3]);
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) p[i] = v[i];
    }
}

// Lanes of a head: one for 4 elements of each half.
constexpr int append_lanes(int hd) { return hd == 96 ? 16 : hd == 192 ? 32 : hd / 8; }

// A lane holds 4 elements of a head and the 4 that the rotation pairs them
// with, half a head further. Each value is computed in 64 bits and rounded to
// f32 once: what is stored then does not depend on an order of operations,
// and a 4-bit code next to a border is the formula's. Bound by memory: 4
// bytes in and out an element of q, 4 in and half a byte or 2 out of k and v
// (2001 rows of 64 + 8 + 8 heads of 64 into MXFP4: 75 MB in 23 us = 3.3 TB/s;
// with the halves of a pair in two lanes, twice the 64-bit work, 27.5). One
// row: 3 us, the chain from its sequence to its page; the row's values are on
// their way meanwhile. TREE: the rotation is that of the row's depth, which a
// wave counts by joining paths (six steps of two exchanges at most), its parents
// on their way from the start too: 16 rows of 64 + 8 + 8 heads 4.3 us, 64 trees
// of up to 8 rows (f16, 32 + 4 + 4 of 128, norms) 8.8 us = 1.9 TB/s.
template <int DT, int HD, bool TREE>
__global__ void __launch_bounds__(64 * kWaves) k_kv_append(AppendArgs A) {
    constexpr int LANES = append_lanes(HD), HEADS = 64 * kWaves / LANES, half = HD / 2;
    const int row = blockIdx.x, j = threadIdx.x % LANES, hu = blockIdx.y * HEADS + threadIdx.x / LANES;
    const bool live = hu < A.nh + 2 * A.c.nkv && 4 * j < half;
    const int kind = hu < A.nh ? 0 : hu < A.nh + A.c.nkv ? 1 : 2, head = kind == 0 ? hu : kind == 1 ? hu - A.nh : hu - A.nh - A.c.nkv;
    const float *bias = kind == 0 ? A.bq : kind == 1 ? A.bk : A.bv, *norm = kind == 0 ? A.qn : kind == 1 ? A.kn : nullptr;
    const int e = live ? 4 * j : 0;   // of the first half
    float f[8] = {}, g[8] = {};
    double u[8];
    if (live) {   // (on their way while the row's sequence and place are looked up)
        const float *x = (kind == 0 ? A.q + (int64_t)row * A.ldq : kind == 1 ? A.k + (int64_t)row * A.ldk : A.v + (int64_t)row * A.ldv) + head * HD + e;
        load4(x, f);
        load4(x + half, f + 4);
        if (bias) {
            load4(bias + head * HD + e, g);
            load4(bias + head * HD + e + half, g + 4);
        }
    }
    int parent = -1;
    if constexpr (TREE) {
        const int r = row - 63 + (int)(threadIdx.x & 63);
        if (r >= 0) parent = A.parent[r];
    }
    int seq = 0;
    KvSeq sq{};
    if (!find_row<TREE>(A.b, A.c.shift, row, &seq, &sq, A.err)) return;
    const int tok = sq.len - sq.n + (row - sq.r0);
    if (tok < 0) return;
    const int page = A.b.pages[(int64_t)seq * A.b.max_pages + (tok >> A.c.shift)];
    int pos = tok;
    if constexpr (TREE) pos = sq.len - sq.n + kv_depth(parent, sq, row, A.err);
    if (A.co && pos >= A.ctx) {
        raise_err(A.err);
        return;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) u[i] = bias ? (double)f[i] + (double)g[i] : (double)f[i];
    if (norm) {   // (the same for the lanes of a head)
        double ss = 0.0;
        if (live)
#pragma unroll
            for (int i = 0; i < 8; ++i) ss = __builtin_fma(u[i], u[i], ss);
#pragma unroll
        for (int o = LANES / 2; o; o >>= 1) ss += __shfl_xor(ss, o, 64);
        const double inv = 1.0 / sqrt(ss / HD + (double)A.eps);
        load4(norm + e, g);
        load4(norm + e + half, g + 4);
#pragma unroll
        for (int i = 0; i < 8; ++i) u[i] = u[i] * inv * (double)g[i];
    }
    if (A.co && kind < 2 && live) {
        load4(A.co + (int64_t)pos * half + e, g);
        load4(A.si + (int64_t)pos * half + e, g + 4);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const double a = u[i], b = u[i + 4], c = g[i], s = g[i + 4];
            u[i] = __builtin_fma(a, c, -b * s);
            u[i + 4] = __builtin_fma(b, c, a * s);
        }
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = (float)u[i];
    // the largest magnitudes (their bits) of the blocks of 32 that the two quads lie in
    int top[2] = {0, 0};
    if constexpr (DT == MH_KV_MXFP4) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
#pragma unroll
            for (int i = 0; i < 4; ++i) top[h] = max(top[h], (int)(__float_as_uint(f[4 * h + i]) & 0x7fffffffu));
            top[h] = max(top[h], __shfl_xor(top[h], 1, 64));
            top[h] = max(top[h], __shfl_xor(top[h], 2, 64));   // 16 elements
        }
        if constexpr (half % 32 == 0) {
#pragma unroll
            for (int h = 0; h < 2; ++h) top[h] = max(top[h], __shfl_xor(top[h], 4, 64));
        } else {   // the other 16 elements of a block, counted through the head in sixteens
            constexpr int N = half / 16;
            const int mine = j / 4;
            int both[2];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int other = min((h * N + mine) ^ 1, 2 * N - 1), from = (threadIdx.x & 63) - j + other % N * 4;
                const int a = __shfl(top[0], from, 64), b = __shfl(top[1], from, 64);
                both[h] = max(top[h], other / N ? b : a);
            }
            top[0] = both[0];
            top[1] = both[1];
        }
    }
    if (!live) return;
    if (kind == 0) {
        float *o = A.q_out + ((int64_t)row * A.nh + head) * HD + e;
        store4(o, f);
        store4(o + half, f + 4);
        return;
    }
    if (!kv_page_ok(A.c, page)) {
        raise_err(A.err);
        return;
    }
    const uint64_t slot = kv_slot(A.c, page, head, tok & ((1 << A.c.shift) - 1));
    uint8_t *dst = kind == 1 ? A.c.k : A.c.v, *exps = kind == 1 ? A.c.ks : A.c.vs;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const int at = e + h * half;
        const float *w = f + 4 * h;
        if constexpr (DT == MH_KV_F16) {
            *(uint2 *)(dst + (slot * HD + at) * 2) =
                make_uint2(kv_f16(w[0]) | (uint32_t)kv_f16(w[1]) << 16, kv_f16(w[2]) | (uint32_t)kv_f16(w[3]) << 16);
        } else {
            // the converter rounds x / scale to the nearest code, ties to even, magnitudes beyond 6 to 6
            const int eb = kv_block_exp((uint32_t)top[h]);
            const float sc = eb == 255 ? 1.f : __uint_as_float((uint32_t)eb << 23);
            uint32_t c = 0;
            c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, w[0], w[1], sc, 0);
            c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, w[2], w[3], sc, 1);
            *(uint16_t *)(dst + (slot * HD + at) / 2) = (uint16_t)c;
            if (at % 32 == 0) exps[slot * (HD / 32) + at / 32] = (uint8_t)eb;
        }
    }
}

// The stored values of a row, 8 elements a lane, heads of k then of v. Bound
// by memory: 2001 rows of 8 heads of 64 (9 MB) 4.8 us, one row 1.8.
__global__ void __launch_bounds__(64 * kWaves) k_kv_read(KvCacheDev c, KvBatchDev b, float *ko, float *vo, unsigned *err) {
    const int row = blockIdx.x, hd = c.hd, i = (blockIdx.y * 64 * kWaves + threadIdx.x) * 8, w = c.nkv * hd;
    int seq;
    KvSeq q;
    if (!find_row<false>(b, c.shift, row, &seq, &q, err)) return;
    const int pos = q.len - q.n + (row - q.r0);
    if (pos < 0 || i >= 2 * w) return;
    const bool isv = i >= w;
    float *out = isv ? vo : ko;
    if (!out) return;
    const int at = isv ? i - w : i, head = at / hd, e = at - head * hd;
    const int page = b.pages[(int64_t)seq * b.max_pages + (pos >> c.shift)];
    if (!kv_page_ok(c, page)) {
        raise_err(err);
        return;
    }
    const uint64_t slot = kv_slot(c, page, head, pos & ((1 << c.shift) - 1));
    const uint8_t *src = isv ? c.v : c.k;
    float f[8];
    if (c.dt == MH_KV_F16) {
        const uint4 r = *(const uint4 *)(src + (slot * hd + e) * 2);
        const uint32_t h[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
        for (int n = 0; n < 4; ++n) {
            f[2 * n] = mh_f16((uint16_t)h[n]);
            f[2 * n + 1] = mh_f16((uint16_t)(h[n] >> 16));
        }
    } else {
        const uint32_t r = *(const uint32_t *)(src + (slot * hd + e) / 2);
        const float sc = __uint_as_float((uint32_t)(isv ? c.vs : c.ks)[slot * (hd / 32) + e / 32] << 23);   // (byte 255: NaN)
        const mh_v2f p0 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(r, sc, 0), p1 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(r, sc, 1);
        const mh_v2f p2 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(r, sc, 2), p3 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(r, sc, 3);
        f[0] = p0.x, f[1] = p0.y, f[2] = p1.x, f[3] = p1.y, f[4] = p2.x, f[5] = p2.y, f[6] = p3.x, f[7] = p3.y;
    }
    float *o = out + (int64_t)row * w + at;
    if ((uintptr_t)o % 16 == 0) {
        ((float4 *)o)[0] = make_float4(f[0], f[1], f[2], f[3]);
        ((float4 *)o)[1] = make_float4(f[4], f[5], f[6], f[7]);
    } else {
#pragma unroll
        for (int n = 0; n < 8; ++n) o[n] = f[n];
    }
}

template <int DT, int HD, bool TREE>
void append_launch(const AppendArgs &A) {
    constexpr int HEADS = 64 * kWaves / append_lanes(HD);
    const unsigned parts = (unsigned)((A.nh + 2 * A.c.nkv + HEADS - 1) / HEADS);
    MH_LAUNCH("kv_append", (k_kv_append<DT, HD, TREE>), dim3((unsigned)A.b.n_rows, parts), dim3(64 * kWaves), 0, stream(), A);
}

template <int DT, bool TREE>
void append_hd(const AppendArgs &A) {
    switch (A.c.hd) {
    case 32: return append_launch<DT, 32, TREE>(A);
    case 64: return append_launch<DT, 64, TREE>(A);
    case 96: return append_launch<DT, 96, TREE>(A);
    case 128: return append_launch<DT, 128, TREE>(A);
    case 192: return append_launch<DT, 192, TREE>(A);
    }
    return append_launch<DT, 256, TREE>(A);
}

}  // namespace

// Checks, resolution and launch of both entry points.
static int append(const mh_kv_cache *c, const mh_kv_batch *b, bool tree, const int32_t *parent, const mh_kv_rows *r, const char *what) {
    clear_error();
    MH_TRY(kv_validate(c, b, what));
    if (tree) MH_TRY(kv_tree_validate(b, parent, what));
    if (!r || !r->q || !r->k || !r->v || !r->q_out) return fail(MH_E_ARG, "%s: NULL rows", what);
    const int hd = c->head_dim, nh = r->n_heads, nkv = c->n_kv_heads;
    if (nh < 1 || nh > 65535 || nh % nkv) return fail(MH_E_ARG, "%s: %d query heads on %d k/v heads", what, nh, nkv);
    const int64_t qd = (int64_t)nh * hd, kvd = (int64_t)nkv * hd;
    const int64_t far = (int64_t)1 << 40;
    if (r->ldq < qd || r->ldk < kvd || r->ldv < kvd || r->ldq > far || r->ldk > far || r->ldv > far)
        return fail(MH_E_ARG, "%s: rows of %lld, %lld, %lld floats do not hold the heads", what, (long long)r->ldq, (long long)r->ldk,
                    (long long)r->ldv);
    if (!r->rope_cos != !r->rope_sin) return fail(MH_E_ARG, "%s: one rotation table without the other", what);
    if (r->rope_cos && r->ctx < 1) return fail(MH_E_ARG, "%s: rotation tables of %d positions", what, r->ctx);
    if (!(r->norm_eps >= 0.f) && (r->qn || r->kn)) return fail(MH_E_ARG, "%s: norm_eps %g", what, (double)r->norm_eps);
    if (((uintptr_t)r->q | (uintptr_t)r->k | (uintptr_t)r->v | (uintptr_t)r->q_out) % 4) return fail(MH_E_ARG, "%s: misaligned rows", what);
    AppendArgs A{};
    const struct {
        const float *p;
        uint64_t bytes;
        const float **to;
    } w[] = {{r->bq, 4 * (uint64_t)qd, &A.bq}, {r->bk, 4 * (uint64_t)kvd, &A.bk}, {r->bv, 4 * (uint64_t)kvd, &A.bv},
             {r->qn, 4 * (uint64_t)hd, &A.qn}, {r->kn, 4 * (uint64_t)hd, &A.kn},
             {r->rope_cos, 2 * (uint64_t)r->ctx * hd, &A.co}, {r->rope_sin, 2 * (uint64_t)r->ctx * hd, &A.si}};
    for (const auto &t : w)
        if ((uintptr_t)t.p % 4) return fail(MH_E_ARG, "%s: a misaligned bias, norm weight or table", what);
    uint64_t qb, kb, vb;
    const uint64_t ob = 4 * (uint64_t)b->n_rows * qd;
    MH_TRY(rows_bytes(b->n_rows, r->ldq, qd, &qb, what));
    MH_TRY(rows_bytes(b->n_rows, r->ldk, kvd, &kb, what));
    MH_TRY(rows_bytes(b->n_rows, r->ldv, kvd, &vb, what));
    if (b->n_rows) {
        if (!(r->q_out == r->q && r->ldq == qd) && kv_overlap(r->q_out, ob, r->q, qb))
            return fail(MH_E_ARG, "%s: q_out overlaps q (it may be q itself where ldq is the heads' width)", what);
        if (tree && kv_overlap(r->q_out, ob, parent, 4 * (uint64_t)b->n_rows)) return fail(MH_E_ARG, "%s: q_out overlaps parent", what);
        if (kv_overlap(r->q_out, ob, r->k, kb) || kv_overlap(r->q_out, ob, r->v, vb)) return fail(MH_E_ARG, "%s: q_out overlaps k or v", what);
        for (const auto &t : w)
            if (t.p && kv_overlap(r->q_out, ob, t.p, t.bytes)) return fail(MH_E_ARG, "%s: q_out overlaps a bias, norm weight or table", what);
    }
    MH_TRY(require_init());
    if (!b->n_rows) return MH_OK;
    OnDevice here;
    MH_TRY(kv_resolve(c, b, &A.c, &A.b, what));
    MH_TRY(resolve_here(r->q, qb, what));
    MH_TRY(resolve_here(r->k, kb, what));
    MH_TRY(resolve_here(r->v, vb, what));
    MH_TRY(resolve_here(r->q_out, ob, what));
    MH_TRY(kv_apart(c, b, r->q_out, ob, what));
    MH_TRY(kv_apart(c, b, r->q, qb, what));   // (the call writes the cache)
    MH_TRY(kv_apart(c, b, r->k, kb, what));
    MH_TRY(kv_apart(c, b, r->v, vb, what));
    const uint64_t cb = kv_cache_bytes(c);
    if (kv_overlap(c->k, cb, c->v, cb) || (c->dt == MH_KV_MXFP4 && (kv_overlap(c->ks, cb / 16, c->vs, cb / 16) || kv_overlap(c->ks, cb / 16, c->k, cb) ||
                                           kv_overlap(c->ks, cb / 16, c->v, cb) || kv_overlap(c->vs, cb / 16, c->k, cb) || kv_overlap(c->vs, cb / 16, c->v, cb))))
        return fail(MH_E_ARG, "%s: the cache's k and v overlap", what);
    if (b->row0) MH_TRY(apart_from_cache(c, b->row0, 4 * ((uint64_t)b->n_seqs + 1), what));
    if (tree) {
        MH_TRY(kv_tree_resolve(b, parent, what));
        MH_TRY(apart_from_cache(c, parent, 4 * (uint64_t)b->n_rows, what));
    }
    MH_TRY(apart_from_cache(c, b->len, 4 * (uint64_t)b->n_seqs, what));
    MH_TRY(apart_from_cache(c, b->pages, 4 * (uint64_t)b->n_seqs * b->max_pages, what));
    for (const auto &t : w)
        if (t.p) {
            const void *d;
            MH_TRY(resolve_weight(t.p, t.bytes, &d, what, true));
            MH_TRY(apart_from_cache(c, d, t.bytes, what));
            if (kv_overlap(r->q_out, 4 * (uint64_t)b->n_rows * qd, d, t.bytes))   // (a region's device copy)
                return fail(MH_E_ARG, "%s: q_out overlaps a bias, norm weight or table", what);
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
    A.parent = parent;
    if (c->dt == MH_KV_F16) tree ? append_hd<MH_KV_F16, true>(A) : append_hd<MH_KV_F16, false>(A);
    else tree ? append_hd<MH_KV_MXFP4, true>(A) : append_hd<MH_KV_MXFP4, false>(A);
    return hip_check(hipGetLastError(), "kv append launch");
}

// mh_kv_check and mh_kv_tree_check.
static int check(const mh_kv_cache *c, const mh_kv_batch *b, bool tree, const int32_t *parent, const char *what) {
    clear_error();
    MH_TRY(kv_validate(c, b, what));
    if (tree) MH_TRY(kv_tree_validate(b, parent, what));
    KvCacheDev cd{};
    cd.n_pages = c->n_pages;
    const int shift = __builtin_ctz((unsigned)c->page);
    const KvBatchDev bd{b->row0, b->len, b->pages, b->n_seqs, b->n_rows, b->max_rows, b->max_pages};
    for (int s = 0; s < b->n_seqs; ++s) {
        KvSeq q;
        if (!(tree ? kv_tree_seq(bd, shift, s, &q) : kv_seq(bd, shift, s, &q)))
            return fail(MH_E_RANGE, "%s: sequence %d: rows %d + %d of %d (at most %d), %d tokens on %d pages", what, s, q.r0, q.n,
                        b->n_rows, b->max_rows, q.len, b->max_pages);
        for (int64_t t = 0; t < q.len; t += c->page) {
            const int p = b->pages[(int64_t)s * b->max_pages + (t >> shift)];
            if (!kv_page_ok(cd, p))
                return fail(MH_E_RANGE, "%s: sequence %d: page %d of %lld holds token %lld", what, s, p, (long long)c->n_pages, (long long)t);
        }
        for (int i = 0; tree && i < q.n; ++i)
            if (parent[q.r0 + i] < -1 || parent[q.r0 + i] >= i)
                return fail(MH_E_RANGE, "%s: sequence %d: row %d follows row %d", what, s, i, parent[q.r0 + i]);
    }
    return MH_OK;
}

}  // namespace mh

using namespace mh;

extern "C" {

int mh_kv_append_dev(const mh_kv_cache *c, const mh_kv_batch *b, const mh_kv_rows *r) {
    return append(c, b, false, nullptr, r, "mh_kv_append_dev");
}

int mh_kv_tree_append_dev(const mh_kv_cache *c, const mh_kv_batch *b, const int32_t *parent, const mh_kv_rows *r) {
    return append(c, b, true, parent, r, "mh_kv_tree_append_dev");
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
    for (const float *p : {k, v})
        if (p) {
            MH_TRY(resolve_here(p, bytes, what));
            MH_TRY(kv_apart(c, b, p, bytes, what));
        }
    unsigned *err;
    MH_TRY(kv_flag(&err));
    const unsigned parts = (unsigned)((2 * c->n_kv_heads * c->head_dim + 64 * kWaves * 8 - 1) / (64 * kWaves * 8));
    MH_LAUNCH("kv_read", k_kv_read, dim3((unsigned)b->n_rows, parts), dim3(64 * kWaves), 0, stream(), cd, bd, k, v, err);
    return hip_check(hipGetLastError(), "kv read launch");
}

int mh_kv_check(const mh_kv_cache *c, const mh_kv_batch *b) { return check(c, b, false, nullptr, "mh_kv_check"); }

int mh_kv_tree_check(const mh_kv_cache *c, const mh_kv_batch *b, const int32_t *parent) {
    return check(c, b, true, parent, "mh_kv_tree_check");
}

}  // extern "C"
