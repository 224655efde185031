// mh_kvattn.hip — attention of a batch's rows over a paged k/v cache
// (mh_kv_attention_dev): attention()'s scores, softmax and weighted sum
// (engine/midge.c:371-396) for many sequences, from f16 or MXFP4.
#include "mh_kvattn.cuh"

namespace mh {
namespace {

// Four elements of a row's result: the weighted sum over the weights' sum
// and the sink's, both in units of 2^(M - kBias); zero for a row before the
// sequence's first token.
template <int HD>
__device__ __forceinline__ void few_out(const KvAttnArgs &A, const KvSeq &q, int row, int h, int d, kv_f4 v, float M, float L) {
    if (A.sink) L += __builtin_amdgcn_exp2f(A.sink[h] * 1.44269504088896341f - (M - kBias));
    v /= L;
    if (q.len - q.n + row < 0) v = kv_f4{0.f, 0.f, 0.f, 0.f};
    *(kv_f4 *)&A.out[((int64_t)(q.r0 + row) * A.nh + h) * HD + d] = v;
}

// ------------------------------------------------- few columns a sequence
//
// A decode step: the columns of a sequence and k/v head are its rows x the
// heads of the group (8 for one token of 64 heads on 8), and the cache is
// read once. Work units are quanta of QT tokens of a (sequence, k/v head);
// the units of all sequences in one line are cut into equal parts, one a
// block, wherever the cuts fall (a block may end one sequence and begin the
// next). The four waves of a block take tiles of the quantum in turn, each
// with its own running softmax, and are joined in LDS where the segment
// ends; a segment that a cut divides is joined by k_kv_join from partial
// results.
//
// A tile: S^T = K Q^T with tokens as the rows of 16x16x32 products and the
// columns (rows x heads) as theirs, so that a lane's scores are those of one
// column, and four consecutive tokens of each 16 are in its registers: as
// they stand they are the second operand of O^T = V^T P^T under the token
// order {4 g + r, 16 + 4 g + r} of a lane group g, which V^T follows. V rows go
// through LDS as f16 and come back transposed (tr16 reads). q and the
// weights are two f16 terms each. Up to 8 columns (NT = 0) the two terms of q
// are stacked in one operand's 16 columns: the score is the sum of columns c
// and c + 8, which a row rotation gives to both, the weights' terms are
// stacked alike, and the second terms cost no instruction. Beyond, NT = 1, 2, 4
// operands of 16 columns, twice the products.
//
// More than 16 columns: MXFP4 rows are few bytes, and the registers are the
// limit, so NT waves take the same tile, 16 columns each (32 columns on 4 k/v
// heads of 128, 32 sequences of 4000 tokens: 45 us; two operands in a wave
// 50). f16 rows are the limit themselves: a wave keeps two operands (the
// same 60 us; two waves 78), unless they no longer fit its registers (of 256:
// 195 us; two waves 79).
//
// Bound by the cache's bytes where there are many: 16 sequences of 500 to 8191
// tokens (f16, 32 heads on 8 of 128) 47 us = 4.0 TB/s. From 4 bits it is not:
// one of 131071 (MXFP4, 64 heads on 8 of 64) 24 us = 3.0 TB/s, 32 of 100 to
// 16000 of the same 27 us = 2.1 TB/s, 4 rows on 32 of 4000 (4 heads of 128) 42
// us = 1.8 TB/s, where a wave's loads, conversions and products follow one
// another and its registers hold no second tile. (Tiles on their way in LDS,
// past the registers, were not tried.) Where there are few bytes, by the chain
// of loads (lengths, page, rows, q, result): one of 4100 tokens 7 us.
template <int DT, int HD, int NT>
struct KvFew {
    using R = KvRow<DT, HD>;
    // operands of 16 columns in all: NC in a wave, CG waves on the same tile; TW tiles at once
    static constexpr int NC = DT == MH_KV_F16 && HD <= 128 && NT > 1 ? 2 : 1, CG = NT ? NT / NC : 1, TW = 4 / CG, COLS = NT ? 16 * NT : 8;
    static constexpr int NS = DT == MH_KV_F16 || HD == 256 ? 2 : 4;   // 16-token parts of a tile
    static constexpr int TILE = 16 * NS, QT = TW * TILE;
    static constexpr int VROW = HD + 16;                              // f16 of a V row in LDS (no bank twice in 8 rows)
    static constexpr int SLOT = COLS * (HD + 2);                      // floats of a partial result
    // waves a SIMD that the registers allow without spilling (LDS allows as many blocks a CU), all resident at once:
    // with 2 or 3 blocks a CU where 4 fit, 32 sequences of MXFP4 of 64 take 42 and 34 us rather than 29.5
    static constexpr int WAVES = HD <= 64 ? (NC == 1 ? 4 : 2) : HD == 96 ? (NC == 1 ? 3 : 2) : HD == 128 ? (NT == 0 && DT != MH_KV_F16 ? 3 : NC == 1 ? 2 : 1) : NT == 0 && DT != MH_KV_F16 ? 2 : 1;
};

// The units of sequence s: QT tokens from the 64 that hold the first token
// which any of its rows sees; one unit if it has rows but no tokens.
__device__ __forceinline__ int few_units(const KvAttnArgs &A, int QT, int s, KvSeq *q, int *a) {
    if (!kv_seq(A.b, A.c.shift, s, q)) {
        raise_err(A.err);
        return 0;
    }
    if (!q->n) return 0;
    const int p0 = max(q->len - q->n, 0), lo = A.window > 0 ? max(0, p0 + 1 - A.window) : 0;
    *a = lo & ~63;
    return max(1, (q->len - *a + QT - 1) / QT);
}

// Inclusive sum over the block's threads in order (256 threads).
__device__ __forceinline__ int block_scan(int v, int *lds) {
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const int u = __shfl_up(v, o, 64);
        if (lane >= o) v += u;
    }
    __syncthreads();
    if (lane == 63) lds[w] = v;
    __syncthreads();
    for (int i = 0; i < w; ++i) v += lds[i];
    return v;
}

// The block's part [*u, *end) of the Q units of the batch, the sequence that
// holds *u and its first unit; block 0 leaves every sequence's first unit
// (and Q) in plan.
__device__ __forceinline__ int64_t few_plan(const KvAttnArgs &A, int QT, int64_t *plan, int64_t *u, int64_t *end, int *seq, int64_t *base) {
    __shared__ int lds[4];
    __shared__ int64_t found[2];
    const int t = threadIdx.x, nkv = A.c.nkv, n = A.b.n_seqs;
    int64_t Q = 0;
    KvSeq q;
    int a;
    if (n == 1) {
        Q = (int64_t)few_units(A, QT, 0, &q, &a) * nkv;
        found[0] = found[1] = 0;
    }
    const int last = n == 1 ? 0 : n;
    for (int pass = n > 256 ? 0 : 1; pass < 2; ++pass) {
        int64_t at = 0;
        for (int c = 0; c < last; c += 256) {
            const int mine = c + t < n ? few_units(A, QT, c + t, &q, &a) : 0, incl = block_scan(mine, lds);
            __shared__ int sum;
            if (t == 255) sum = incl;
            __syncthreads();
            if (n <= 256) Q = (int64_t)sum * nkv;
            if (pass) {
                const int64_t first = (at + incl - mine) * nkv, g = min((int64_t)A.grid, Q);
                const int64_t start = g ? kv_div((int64_t)blockIdx.x * Q, g) : 0;
                if (mine && start >= first && start < first + (int64_t)mine * nkv) {
                    found[0] = c + t;
                    found[1] = first;
                }
                if (blockIdx.x == 0 && c + t < n) plan[c + t] = first;
            }
            at += sum;
            __syncthreads();
        }
        if (n > 256 && !pass) Q = at * nkv;
    }
    if (blockIdx.x == 0 && t == 0) {
        plan[n] = Q;
        if (n == 1) plan[0] = 0;
    }
    __syncthreads();
    const int64_t g = min((int64_t)A.grid, Q);
    if ((int64_t)blockIdx.x >= g) return 0;
    *u = kv_div((int64_t)blockIdx.x * Q, g);
    *end = kv_div(((int64_t)blockIdx.x + 1) * Q, g);
    *seq = (int)found[0];
    *base = found[1];
    return Q;
}

template <int DT, int HD, int NT>
__global__ void __launch_bounds__(256, (KvFew<DT, HD, NT>::WAVES)) k_kv_few(KvAttnArgs A, int64_t *plan) {
    using F = KvFew<DT, HD, NT>;
    using R = KvRow<DT, HD>;
    constexpr int NC = F::NC, TW = F::TW, COLS = F::COLS, ROUND = COLS / NC, NS = F::NS, TILE = F::TILE, VROW = F::VROW, SPC = R::CH / 8;
    __shared__ __attribute__((aligned(16))) _Float16 vbuf[4][32 * VROW];
    __shared__ float sm[TW][COLS], sl[TW][COLS];
    float *const mb = (float *)&vbuf[0][0];   // the waves' results once a segment's tiles are done
    static_assert(TW * ROUND * HD * 4 <= sizeof(vbuf), "the waves' results lie in V's rows");
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, t = lane & 15, g = lane >> 4;
    const int tw = wave % TW, cg = wave / TW, c0 = NT ? 16 * cg + t : t & 7;   // this lane's columns: c0 + n * ROUND
    int64_t u, end, base;
    int seq;
    if (!few_plan(A, F::QT, plan, &u, &end, &seq, &base)) return;
    const int64_t u0 = u;
    _Float16 *const vt = vbuf[wave];
    const uint32_t off = KvFrag<DT, HD>::lane_off(t, g), eoff = KvFrag<DT, HD>::lane_eoff(t, g);
    while (u < end && seq < A.b.n_seqs) {
        KvSeq q;
        int a = 0;
        const int nq = few_units(A, F::QT, seq, &q, &a);
        if (nq == 0) {   // (a sequence without rows)
            ++seq;
            continue;
        }
        const int head = (int)kv_div(u - base, nq), qi = (int)(u - base - (int64_t)head * nq);
        const int qe = (int)min((int64_t)nq, qi + (end - u));
        const int cols = q.n * A.group;
        kv_h8 qa[NC][R::KS], qb[NT ? NC : 1][R::KS];
        float inv[NC], m[NC], ms[NC], l[NC];
        int pos[NC];
        const bool first_term = NT != 0 || t < 8;
        const float part = first_term ? 0.f : -1.f, minus = kv_minus();
#pragma unroll
        for (int n = 0; n < NC; ++n) {
            const int c = c0 + n * ROUND;
            pos[n] = c < cols ? max(q.len - q.n + c / A.group, -1) : -1;
            inv[n] = 1.f;
            m[n] = -INFINITY;
            ms[n] = -kBias;
            l[n] = 0.f;
#pragma unroll
            for (int k = 0; k < R::KS; ++k) {
                qa[n][k] = kv_h8{0};
                if constexpr (NT != 0) qb[n][k] = kv_h8{0};
            }
        }
        // the columns' q as matrix operands: (q * qscale) * 2^(13 - exponent of the row's largest)
        auto make_q = [&]() KV_INLINE {
#pragma unroll
            for (int n = 0; n < NC; ++n) {
                const int c = c0 + n * ROUND;
                const bool ok = c < cols;
                const int row = ok ? c / A.group : 0;
                const float *src = A.q + ((int64_t)(q.r0 + row) * A.nh + head * A.group + (ok ? c - row * A.group : 0)) * HD;
                float x[R::KS][8], mx = 0.f;
#pragma unroll
                for (int i = 0; i < R::NL; ++i)
#pragma unroll
                    for (int s = 0; s < SPC; ++s) {
                        const float4 *p = (const float4 *)(src + 4 * R::CH * i + R::CH * g + 8 * s);
                        const float4 v0 = p[0], v1 = p[1];
                        const float v[8] = {v0.x, v0.y, v0.z, v0.w, v1.x, v1.y, v1.z, v1.w};
#pragma unroll
                        for (int e = 0; e < 8; ++e) {
                            x[i * SPC + s][e] = ok ? v[e] * A.qscale : 0.f;
                            mx = fmaxf(mx, fabsf(x[i * SPC + s][e]));
                        }
                    }
                mx = fmaxf(mx, __shfl_xor(mx, 16, 64));
                mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
                const int ex = min(max((int)(__float_as_uint(mx) >> 23) - 126, -100), 128);
                const float up = __uint_as_float((uint32_t)(13 - ex + 127) << 23);
                inv[n] = __uint_as_float((uint32_t)(ex - 13 + 127) << 23);
#pragma unroll
                for (int k = 0; k < R::KS; ++k)
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        _Float16 hi, lo;
                        kv_split(x[k][e] * up, &hi, &lo);
                        if constexpr (NT == 0) {
                            qa[n][k][e] = t >= 8 ? lo : hi;
                        } else {
                            qa[n][k][e] = hi;
                            qb[n][k][e] = lo;
                        }
                    }
            }
        };
        kv_f4 o[NC][HD / 16];
#pragma unroll
        for (int n = 0; n < NC; ++n)
#pragma unroll
            for (int d = 0; d < HD / 16; ++d) o[n][d] = kv_f4{0.f, 0.f, 0.f, 0.f};
        const int first = q.len - q.n + 1;                                      // tokens that the first row sees
        const int lo_all = A.window > 0 ? max(0, q.len - A.window) : 0;           // from here on the last row does
        const int lo_any = A.window > 0 ? max(0, max(first, 1) - A.window) : 0;
        const int32_t *pages = A.b.pages + (int64_t)seq * A.b.max_pages;
        bool ready = false;
        for (int i4 = 16 * cg < cols ? qi : qe; i4 < qe; ++i4) {   // (no tiles for a wave past the last column)
            const int t0 = a + i4 * F::QT + tw * TILE;
            if (t0 >= q.len) break;
            KvFrag<DT, HD> kf[NS], vf[NS];
            bool bad[NS], anybad = false;
#pragma unroll
            for (int j = 0; j < NS; ++j) {
                const int tok = t0 + 16 * j;
                const int page = kv_word(pages, min(tok, q.len - 1) >> A.c.shift);
                const bool valid = kv_page_ok(A.c, page);
                bad[j] = !valid && tok + 16 > lo_any;   // (behind every row's window a page may be anything)
                anybad |= bad[j];
                const uint64_t slot = kv_slot(A.c, valid ? page : 0, head, tok & ((1 << A.c.shift) - 1));
                kf[j].load(A.c.k + slot * R::ROW, A.c.ks + slot * (HD / 32), off, eoff);
                vf[j].load(A.c.v + slot * R::ROW, A.c.vs + slot * (HD / 32), off, eoff);
            }
            if (anybad) raise_err(A.err);
            if (!ready) {   // (while the first rows are on their way)
                make_q();
                ready = true;
            }
            // the tiles at the ends, and those with a page out of bounds: what the columns do not see
            const int edge = __builtin_amdgcn_readfirstlane(t0 + TILE > first || t0 < lo_all || anybad);
            int oddm = 0;
            // (loops of one pass or none, with an operand that is new in each: as branches they become selects
            // in every tile)
            int pass = edge;
            asm volatile("" : "+s"(pass));
            for (; pass; --pass) {
                int tok = t0 + t;
                asm volatile("" : "+v"(tok));
#pragma unroll
                for (int j = 0; j < NS; ++j) {
                    if (tok + 16 * j >= q.len || tok + 16 * j < lo_any) vf[j].zero();   // whatever a stale slot holds
                    if (q.n > 1) {
                        bool odd = false;
#pragma unroll
                        for (int i = 0; i < R::NL; ++i)
#pragma unroll
                            for (int k = 0; k < SPC; ++k) odd |= kv_odd(vf[j].eight(i, k));
                        oddm |= (__ballot(odd) != 0) << (j / 2);
                    }
                }
            }
            kv_f4 s[NC][NS];
#pragma unroll
            for (int j = 0; j < NS; ++j) {
#pragma unroll
                for (int n = 0; n < NC; ++n) s[n][j] = kv_f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int i = 0; i < R::NL; ++i)
#pragma unroll
                    for (int k = 0; k < SPC; ++k) {
                        const kv_h8 kk = kf[j].eight(i, k);
#pragma unroll
                        for (int n = 0; n < NC; ++n) {
                            if constexpr (NT != 0)
                                s[n][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kk, qb[n][i * SPC + k], s[n][j], 0, 0, 0);
                            s[n][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kk, qa[n][i * SPC + k], s[n][j], 0, 0, 0);
                        }
                    }
            }
            float tm[NC];
            auto largest = [&]() {
#pragma unroll
                for (int n = 0; n < NC; ++n) {
                    float x = -INFINITY;
#pragma unroll
                    for (int j = 0; j < NS; ++j) x = fmaxf(fmaxf(fmaxf(x, s[n][j][0]), s[n][j][1]), fmaxf(s[n][j][2], s[n][j][3]));
                    tm[n] = x * inv[n];
                }
            };
            if constexpr (NT == 0)
#pragma unroll
                for (int j = 0; j < NS; ++j)
#pragma unroll
                    for (int r = 0; r < 4; ++r) s[0][j][r] += kv_ror8(s[0][j][r]);
            largest();
            pass = edge;
            asm volatile("" : "+s"(pass));
            for (; pass; --pass) {
                int tok = t0 + 4 * g;
                asm volatile("" : "+v"(tok));
                const uint32_t w = A.window > 0 ? (uint32_t)A.window : (uint32_t)INT32_MAX;
#pragma unroll
                for (int n = 0; n < NC; ++n)
#pragma unroll
                    for (int j = 0; j < NS; ++j)
#pragma unroll
                        for (int r = 0; r < 4; ++r)   // 0 <= pos - token < window
                            s[n][j][r] = (uint32_t)(pos[n] - tok) - (uint32_t)(16 * j + r) < w ? (bad[j] ? NAN : s[n][j][r]) : -INFINITY;
                largest();
            }
            bool up = false;
#pragma unroll
            for (int n = 0; n < NC; ++n) up |= tm[n] > m[n] + kLag;
            if (__ballot(up)) {
#pragma unroll
                for (int n = 0; n < NC; ++n) {
                    float x = fmaxf(tm[n], __shfl_xor(tm[n], 16, 64));
                    x = fmaxf(x, __shfl_xor(x, 32, 64));
                    const float mn = fmaxf(m[n], x);
                    const float al = mn == m[n] ? 1.f : __builtin_amdgcn_exp2f(m[n] - mn);
                    m[n] = mn;
                    ms[n] = mn == -INFINITY ? -kBias : mn - kBias;
                    l[n] *= al;
#pragma unroll
                    for (int d = 0; d < HD / 16; ++d) o[n][d] *= al;
                }
            }
            kv_h8 pa[NC][NS / 2], pb[NT ? NC : 1][NS / 2];
#pragma unroll
            for (int n = 0; n < NC; ++n)
#pragma unroll
                for (int j = 0; j < NS; ++j)
#pragma unroll
                    for (int r = 0; r < 4; r += 2) {
                        const float p0 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[n][j][r], inv[n], -ms[n]));
                        const float p1 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[n][j][r + 1], inv[n], -ms[n]));
                        l[n] += p0;
                        l[n] += p1;
                        const int e = 4 * (j & 1) + r;
                        if constexpr (NT == 0) {   // the first term, or what it leaves
                            const kv_h2 hi = {(_Float16)p0, (_Float16)p1};
                            pa[n][j / 2][e] = (_Float16)__builtin_fmaf((float)hi[0], part, p0);
                            pa[n][j / 2][e + 1] = (_Float16)__builtin_fmaf((float)hi[1], part, p1);
                        } else {
                            kv_h2 hi, lo;
                            kv_split2(p0, p1, minus, &hi, &lo);
                            pa[n][j / 2][e] = hi[0];
                            pa[n][j / 2][e + 1] = hi[1];
                            pb[n][j / 2][e] = lo[0];
                            pb[n][j / 2][e + 1] = lo[1];
                        }
                    }
#pragma unroll
            for (int h = 0; h < NS / 2; ++h) {
#pragma unroll
                for (int jj = 0; jj < 2; ++jj)
#pragma unroll
                    for (int i = 0; i < R::NL; ++i)
#pragma unroll
                        for (int k = 0; k < SPC; ++k)
                            *(kv_h8 *)&vt[(16 * jj + t) * VROW + 4 * R::CH * i + R::CH * g + 8 * k] = vf[2 * h + jj].eight(i, k);
                if (oddm >> h & 1) {
                    // an inf or NaN that some rows see and others do not: token by token, each to
                    // the rows that see it
                    for (int k = 0; k < 32; ++k) {
                        const int tok = t0 + 32 * h + k, from = t + 16 * ((k & 15) >> 2);
#pragma unroll
                        for (int n = 0; n < NC; ++n) {
                            float p = 0.f;
#pragma unroll
                            for (int jj = 0; jj < 2; ++jj)
#pragma unroll
                                for (int r = 0; r < 4; ++r)
                                    p = 16 * jj + r == (k & 19)
                                            ? __builtin_amdgcn_exp2f(__builtin_fmaf(s[n][2 * h + jj][r], inv[n], -ms[n]))
                                            : p;
                            p = __shfl(p, from, 64);
                            const bool sees = tok <= pos[n] && (A.window <= 0 || tok > pos[n] - A.window) && first_term;
#pragma unroll
                            for (int d = 0; d < HD / 16; ++d)
#pragma unroll
                                for (int r = 0; r < 4; ++r) {
                                    const float v = (float)vt[k * VROW + 16 * d + 4 * g + r];
                                    o[n][d][r] = sees ? __builtin_fmaf(p, v, o[n][d][r]) : o[n][d][r];
                                }
                        }
                    }
                    continue;
                }
#pragma unroll
                for (int d = 0; d < HD / 16; ++d) {
                    const _Float16 *p = &vt[(4 * g + (t >> 2)) * VROW + 16 * d + (t & 3) * 4];
                    const kv_h4 v0 = kv_tr16(p), v1 = kv_tr16(p + 16 * VROW);
                    const kv_h8 v = {v0[0], v0[1], v0[2], v0[3], v1[0], v1[1], v1[2], v1[3]};
#pragma unroll
                    for (int n = 0; n < NC; ++n) {
                        if constexpr (NT != 0) o[n][d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v, pb[n][h], o[n][d], 0, 0, 0);
                        o[n][d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v, pa[n][h], o[n][d], 0, 0, 0);
                    }
                }
            }
        }
        // the four waves' results: one maximum, the sums added in wave order
#pragma unroll
        for (int n = 0; n < NC; ++n) {
            l[n] += __shfl_xor(l[n], 16, 64);
            l[n] += __shfl_xor(l[n], 32, 64);
            if (g == 0 && (NT || t < 8)) {
                sm[tw][c0 + n * ROUND] = m[n];
                sl[tw][c0 + n * ROUND] = l[n];
            }
        }
        __syncthreads();
        auto most = [&](int c) KV_INLINE {
            float M = sm[0][c];
#pragma unroll
            for (int w = 1; w < TW; ++w) M = fmaxf(M, sm[w][c]);
            return M;
        };
#pragma unroll
        for (int n = 0; n < NC; ++n) {
            const int c = c0 + n * ROUND;
            const float f = m[n] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m[n] - most(c));
#pragma unroll
            for (int d = 0; d < HD / 16; ++d)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    if constexpr (NT == 0) o[n][d][r] += kv_ror8(o[n][d][r]);
                    o[n][d][r] *= f;
                }
        }
        // [tile][column][HD], as many columns at a time as the rows' space holds
        const bool whole = qi == 0 && qe == nq;
        float *const slot = A.part + (2 * (uint64_t)blockIdx.x + (u == u0 ? 0 : 1)) * F::SLOT;
#pragma unroll
        for (int n = 0; n < NC; ++n) {
            if (n) __syncthreads();
            if (NT || t < 8)
#pragma unroll
                for (int d = 0; d < HD / 16; ++d) *(kv_f4 *)&mb[(tw * ROUND + c0) * HD + 16 * d + 4 * g] = o[n][d];
            __syncthreads();
            for (int i = threadIdx.x; i < min(ROUND, cols - n * ROUND) * (HD / 4); i += 256) {
                const int cr = i / (HD / 4), c = n * ROUND + cr, d = 4 * (i % (HD / 4));
                const float M = most(c);
                float L = 0.f;
                kv_f4 v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int w = 0; w < TW; ++w) {
                    L += sm[w][c] == -INFINITY ? 0.f : sl[w][c] * __builtin_amdgcn_exp2f(sm[w][c] - M);
                    v += *(const kv_f4 *)&mb[(w * ROUND + cr) * HD + d];
                }
                if (!whole) {
                    *(kv_f4 *)&slot[c * HD + d] = v;
                    if (d == 0) {
                        slot[COLS * HD + 2 * c] = M;
                        slot[COLS * HD + 2 * c + 1] = L;
                    }
                } else {
                    const int row = c / A.group, h = head * A.group + c - row * A.group;
                    few_out<HD>(A, q, row, h, d, v, M, L);
                }
            }
        }
        __syncthreads();
        u += qe - qi;
        if (qe == nq && head == A.c.nkv - 1) {
            ++seq;
            base = u;
        }
    }
}

// Joins the partial results of the segment (blockIdx.x: sequence and k/v
// head) for one column (blockIdx.y): those of the blocks between the cuts
// that it holds, in their order. Bound by one trip to memory behind the plan's
// words: 3 to 6 us, beside the launch, also where no segment is divided (a
// token in a window of 128 on MXFP4 is one unit: all blocks return at once, 4
// of 11 us). Joined by the last block to arrive, on counters that each call
// leaves at zero, a segment would be one block's: 17 parts a head of 4100
// tokens, 128 of 131071. Not tried.
template <int HD, int COLS>
__global__ void __launch_bounds__(256) k_kv_join(KvAttnArgs A, const int64_t *plan, int QT) {
    constexpr int SLOT = COLS * (HD + 2), TD = HD / 4, NG = 256 / TD, AT = 4;
    __shared__ float sM[NG], sL[NG];
    __shared__ kv_f4 acc[NG * TD];
    const int s = blockIdx.x / A.c.nkv, head = blockIdx.x - s * A.c.nkv, c = blockIdx.y, t = threadIdx.x;
    const int64_t Q = plan[A.b.n_seqs], G = min((int64_t)A.grid, Q), seg0 = plan[s], seg1 = plan[s + 1];
    KvSeq q;
    const bool ok = kv_seq(A.b, A.c.shift, s, &q);
    const int nq = (int)kv_div(seg1 - seg0, A.c.nkv);
    if (nq == 0 || !ok || c >= q.n * A.group) return;
    const int64_t qs = seg0 + (int64_t)head * nq, qe = qs + nq;
    const int b0 = (int)kv_div((qs + 1) * G - 1, Q), b1 = (int)kv_div(qe * G - 1, Q);
    if (b0 == b1) return;
    const bool late = kv_div((int64_t)b0 * Q, G) < qs;   // the first block began in an earlier segment
    auto slot = [&](int b) { return A.part + (2 * (uint64_t)b + (b == b0 && late ? 1 : 0)) * SLOT; };
    // thread (group gr, elements 4 d ..): every NG-th partial result, AT of them on their way at once
    const int d = t % TD, gr = t / TD;
    float M = -INFINITY, L = 0.f;
    kv_f4 v = {0.f, 0.f, 0.f, 0.f};
    if (gr < NG) {
        for (int b = b0 + gr; b <= b1; b += AT * NG) {
            float mk[AT], lk[AT], mn = M;
            kv_f4 vk[AT];
#pragma unroll
            for (int k = 0; k < AT; ++k) {
                const float *p = slot(min(b + k * NG, b1));
                mk[k] = p[COLS * HD + 2 * c];
                lk[k] = p[COLS * HD + 2 * c + 1];
                vk[k] = *(const kv_f4 *)&p[c * HD + 4 * d];
            }
#pragma unroll
            for (int k = 0; k < AT; ++k) {
                if (b + k * NG > b1) mk[k] = -INFINITY;
                mn = fmaxf(mn, mk[k]);
            }
            const float f = M == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(M - mn);
            v *= f;
            L *= f;
            M = mn;
#pragma unroll
            for (int k = 0; k < AT; ++k)
                if (b + k * NG <= b1) {   // (a block that saw nothing has zeros, or NaN)
                    const float e = mk[k] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(mk[k] - M);
                    v += vk[k] * e;
                    L += lk[k] * e;
                }
        }
        acc[t] = v;
        if (d == 0) {
            sM[gr] = M;
            sL[gr] = L;
        }
    }
    __syncthreads();
    if (gr != 0) return;
    M = sM[0];
    for (int i = 1; i < NG; ++i) M = fmaxf(M, sM[i]);
    v = kv_f4{0.f, 0.f, 0.f, 0.f};
    L = 0.f;
#pragma unroll
    for (int i = 0; i < NG; ++i) {
        const float f = sM[i] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(sM[i] - M);
        v += acc[i * TD + d] * f;
        L += sL[i] * f;
    }
    const int row = c / A.group;
    few_out<HD>(A, q, row, head * A.group + c - row * A.group, 4 * d, v, M, L);
}

// Blocks that share a decode step's units: as many as are resident at once.
constexpr int kGridMax = 4 * 256;

int few_cols(int columns) { return columns <= 8 ? 8 : columns <= 16 ? 16 : columns <= 32 ? 32 : 64; }   // KvFew::COLS

uint64_t plan_bytes(const mh_kv_batch &b) { return (8 * ((uint64_t)b.n_seqs + 1) + 15) / 16 * 16; }

// The largest sequence's columns, as the host knows them.
int64_t most_columns(const mh_kv_batch &b, int group) { return (int64_t)(b.row0 ? std::min(b.max_rows, std::max(b.n_rows, 1)) : 1) * group; }

uint64_t few_ws(const mh_kv_cache &c, const mh_kv_batch &b, int group) {
    const int64_t columns = most_columns(b, group);
    if (columns > kv_few(c.dt, c.head_dim)) return kv_many_ws(c, b, group);
    return plan_bytes(b) + 2ull * kGridMax * few_cols((int)columns) * (c.head_dim + 2) * 4;
}

template <int DT, int HD, int NT>
int few_launch(KvAttnArgs A, void *ws, int columns) {
    using F = KvFew<DT, HD, NT>;
    int64_t *plan = (int64_t *)ws;
    const int64_t most = (int64_t)A.b.n_seqs * A.c.nkv * ((((int64_t)A.b.max_pages << A.c.shift) + 63) / F::QT + 1);   // units
    A.grid = (int)std::min<int64_t>(std::min(device_cus() * F::WAVES, kGridMax), most);
    MH_LAUNCH("kv_few", (k_kv_few<DT, HD, NT>), dim3((unsigned)A.grid), dim3(256), 0, stream(), A, plan);
    MH_LAUNCH("kv_join", (k_kv_join<HD, F::COLS>), dim3((unsigned)(A.b.n_seqs * A.c.nkv), (unsigned)columns), dim3(256), 0, stream(), A,
              (const int64_t *)plan, F::QT);
    return MH_OK;
}

template <int DT, int HD>
int few_nt(const KvAttnArgs &A, void *ws, int columns) {
    const int f = few_cols(columns);
    if (f == 8) return few_launch<DT, HD, 0>(A, ws, columns);
    if (f == 16) return few_launch<DT, HD, 1>(A, ws, columns);
    if constexpr (DT != MH_KV_F16 || HD <= 128)
        if (f == 64) return few_launch<DT, HD, 4>(A, ws, columns);
    return few_launch<DT, HD, 2>(A, ws, columns);
}

template <int DT>
int few_hd(const KvAttnArgs &A, void *ws, int columns) {
    switch (A.c.hd) {
    case 32: return few_nt<DT, 32>(A, ws, columns);
    case 64: return few_nt<DT, 64>(A, ws, columns);
    case 96: return few_nt<DT, 96>(A, ws, columns);
    case 128: return few_nt<DT, 128>(A, ws, columns);
    case 192: return few_nt<DT, 192>(A, ws, columns);
    }
    return few_nt<DT, 256>(A, ws, columns);
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
    *bytes = few_ws(*c, *b, n_heads / c->n_kv_heads);
    return MH_OK;
}

int mh_kv_attention_dev(const mh_kv_cache *c, const mh_kv_batch *b, int n_heads, int window, float scale, const float *sink,
                        const float *q, float *out, void *ws, uint64_t ws_bytes) {
    const char *what = "mh_kv_attention_dev";
    uint64_t need = 0;
    MH_TRY(mh_kv_attention_ws(c, b, n_heads, &need));
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
    const int64_t columns = most_columns(*b, A.group);
    if (columns <= kv_few(c->dt, c->head_dim)) {
        A.part = (float *)((uint8_t *)ws + plan_bytes(*b));
        MH_TRY(c->dt == MH_KV_F16 ? few_hd<MH_KV_F16>(A, ws, (int)columns) : few_hd<MH_KV_MXFP4>(A, ws, (int)columns));
        return hip_check(hipGetLastError(), "kv attention launch");
    }
    return kv_many_run(*c, *b, A, ws);
}

}  // extern "C"
