// mh_kvprompt.hip — attention of prompt chunks over a paged k/v cache
// (mh_kv_attention_dev where a sequence has more than kv_few() columns).
//
// A segment is 128 columns (rows x heads of the group) of a sequence and k/v
// head; its work units are tiles of TILE tokens, from the first that any of
// its rows sees to the last. k_kv_plan lines up the units of one head over
// all sequences; the heads' lines in one row are cut into equal parts, one a
// block, wherever the cuts fall, and segments that a cut divides are joined
// by k_kv_pjoin. Consecutive parts go to one XCD, whose L2 then holds a
// head's k and v for all of them.
//
// A tile: the four waves bring its rows into LDS as f16, each takes 32
// columns. S^T = K Q^T by 32x32x16 products, so that a lane's scores are those
// of one column; as they stand in its registers they are the second operand
// of O^T = V^T P^T under the token order {16 s + 4 h + j, 16 s + 8 + 4 h + j} of a
// lane half h, which the transposing LDS reads of V follow. q and the weights
// are two f16 terms each: twice the products, 22 bits. The exponentials and
// splits of a tile take about as long as its products: the loop makes the
// scores of tile i + 1 while it makes the weights of tile i, and looks for the
// maximum of tile i + 1 while it adds the values of tile i, so that both run at
// once in every wave. k of tile i + 2 and v of tile i + 1 come in meanwhile,
// their raw rows loaded an iteration earlier: one barrier a tile.
//
// Bound by issue: 4000 tokens of a prompt (MXFP4, 64 heads on 8 of 64) take
// 300 us = 437 TFLOP/s of the formula, 874 of f16 products (a library
// product of 8192^3 on this card: 1171); the matrix cores are busy for 44% of
// the cycles, other vector instructions take 48% and an exponential four
// times as long as those. 512 rows behind 16000 tokens (f16, 32 heads on 4 of
// 128): 277 us, 477 TFLOP/s of the formula. At an
// earlier 305 us: tiles of 32 tokens at 64 elements a row (TT = 1) 340, with 3
// waves a SIMD 310; 3 blocks a CU 337, 4 321. One term of q and of the weights
// would halve the products and leave 11 bits of the scores.
#include "mh_kvattn.cuh"

namespace mh {
namespace {

constexpr int kCols = 128;

template <int DT, int HD>
struct KvMany {
    using R = KvRow<DT, HD>;
    static constexpr int TT = HD <= 64 ? 2 : 1, TILE = 32 * TT;                // (registers: scores of two tiles)
    static constexpr int KROW = HD + 8;                                  // f16 of a K row in LDS: 16-byte reads of 8 rows on 32 banks
    static constexpr int VROW = HD + (HD / 2 % 64 == 16 || HD / 2 % 64 == 48 ? 0 : 32);   // a stride of 16 or 48 banks: 4 rows of 16 apart
    static constexpr int SLOT = kCols * (HD + 2);                        // floats of a partial result
};

// A segment row (128 columns of a sequence): its sequence, its columns' rows and
// the tokens they see.
struct __attribute__((aligned(16))) Row {
    int r0, n, len, seq;       // the sequence (KvSeq)
    int c0, cols, a, nt;       // first column, columns; first token, tiles
    int hi, pad[3];            // end of the tokens
};
// What a segment costs beside its tiles (q, the first rows' latency, the
// result), in tiles: the cuts count it.
constexpr int kExtra = 3;   // (1, 2, 4 and 6: within 1%)
// Segments up to this many tiles are not divided: the block in whose part
// one begins takes all of it (two partial results and their join cost more
// than the tiles: 2000 tokens in a window of 128 take 42 us, divided 49; 4
// and 16 are equal).
constexpr int kWhole = 8;

struct Plan {
    int64_t *up;      // [n_ct + 1]: the first unit of each segment row in one head's line
    Row *row;         // [n_ct]
    int32_t *off;     // [n_seqs + 1]: segment rows before a sequence, at most n_ct
    int32_t *odd;     // [n_kv_heads][n_ct]: segments with an inf or NaN in v that some of their rows do not see
    struct Head {
        int64_t T1;       // units of one head's line
        int32_t nct, any; // segment rows; whether any segment is odd
    } *head;
    struct Info {     // [grid]: the segment that holds a block's first unit
        int64_t qs, qe;   // units of its tiles
        int32_t ct, head;
    } *info;
};

__device__ __forceinline__ Row many_row(const KvAttnArgs &A, const KvSeq &q, int seq, int ct, int TILE) {
    Row z;
    z.r0 = q.r0;
    z.n = q.n;
    z.len = q.len;
    z.seq = seq;
    z.c0 = ct * kCols;
    z.cols = min(kCols, q.n * A.group - z.c0);
    const int ra = z.c0 / A.group, rb = (z.c0 + z.cols - 1) / A.group, pa = max(q.len - q.n + ra, 0);
    z.hi = max(q.len - q.n + rb + 1, 0);
    z.a = (A.window > 0 ? max(0, pa + 1 - A.window) : 0) & -TILE;
    z.nt = max(1, (z.hi - z.a + TILE - 1) / TILE);
    z.pad[0] = z.pad[1] = z.pad[2] = 0;
    return z;
}

template <class T>
__device__ __forceinline__ T scan1024(T v, T *lds, T *total) {
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const T u = __shfl_up(v, o, 64);
        if (lane >= o) v += u;
    }
    __syncthreads();
    if (lane == 63) lds[w] = v;
    __syncthreads();
    T sum = 0;
    for (int i = 0; i < 16; ++i) {
        if (i < w) v += lds[i];
        sum += lds[i];
    }
    *total = sum;
    return v;
}

// One block: up, row and off; odd and any cleared. (4 to 5 us, beside the
// launch; with every block's start found here too, 1 us more and none less
// in k_kv_many.)
__global__ void __launch_bounds__(1024) k_kv_plan(KvAttnArgs A, Plan P, int TILE, int room) {
    __shared__ long long ll[16];
    const int t = threadIdx.x;
    int at = 0;
    for (int s0 = 0; s0 < A.b.n_seqs; s0 += 1024) {
        const int s = s0 + t;
        long long n = 0, sum;
        if (s < A.b.n_seqs) {
            KvSeq q;
            if (kv_seq(A.b, A.c.shift, s, &q)) n = (q.n * A.group + kCols - 1) / kCols;
            else raise_err(A.err);
        }
        // (segment rows past the arrays' room are those of sequences that share rows: left out)
        const long long incl = scan1024(n, ll, &sum);
        if (s < A.b.n_seqs) {
            P.off[s] = (int)min(at + incl - n, (long long)room);
            if (at + incl > room) raise_err(A.err);
        }
        at = (int)min(at + sum, (long long)room);
    }
    if (t == 0) P.off[A.b.n_seqs] = at;
    __threadfence_block();
    __syncthreads();
    long long base = 0;
    for (int c0 = 0; c0 < at; c0 += 1024) {
        const int c = c0 + t;
        long long n = 0, sum;
        if (c < at) {
            int lo = 0, hi = A.b.n_seqs;   // the last sequence whose rows begin at or before c
            while (hi - lo > 1) {
                const int m = (lo + hi) >> 1;
                if (P.off[m] <= c) lo = m;
                else hi = m;
            }
            KvSeq q;
            kv_seq(A.b, A.c.shift, lo, &q);
            const Row z = many_row(A, q, lo, c - P.off[lo], TILE);
            P.row[c] = z;
            n = z.nt + kExtra;
        }
        const long long incl = scan1024(n, ll, &sum);
        if (c < at) P.up[c] = base + incl - n;
        base += sum;
    }
    if (t == 0) {
        P.up[at] = base;
        *P.head = Plan::Head{base, at, 0};
    }
    for (int64_t i = t; i < (int64_t)at * A.c.nkv; i += 1024) P.odd[i] = 0;
}

// Four elements of a row's result (as few_out in mh_kvattn.hip).
template <int HD>
__device__ __forceinline__ void many_out(const KvAttnArgs &A, const Row &q, int col, int head, int d, kv_f4 v, float M, float L) {
    const int row = col / A.group, h = head * A.group + col - row * A.group;
    if (A.sink) L += __builtin_amdgcn_exp2f(A.sink[h] * 1.44269504088896341f - (M - kBias));
    v /= L;
    if (q.len - q.n + row < 0) v = kv_f4{0.f, 0.f, 0.f, 0.f};
    *(kv_f4 *)&A.out[((int64_t)(q.r0 + row) * A.nh + h) * HD + d] = v;
}

// The same for every lane.
__device__ __forceinline__ void uniform(Row &z) {
    for (int *p : {&z.r0, &z.n, &z.len, &z.seq, &z.c0, &z.cols, &z.a, &z.nt, &z.hi}) *p = __builtin_amdgcn_readfirstlane(*p);
}

template <int DT, int HD>
__global__ void __launch_bounds__(256, HD <= 128 ? 2 : 1) k_kv_many(KvAttnArgs A, Plan P) {
    using F = KvMany<DT, HD>;
    using R = KvRow<DT, HD>;
    constexpr int TT = F::TT, TILE = F::TILE, KROW = F::KROW, VROW = F::VROW, SPC = R::CH / 8;
    __shared__ __attribute__((aligned(16))) _Float16 kb[2][TILE * KROW];
    __shared__ __attribute__((aligned(16))) _Float16 vb[2][TILE * VROW];
    __shared__ int fbad[2][4];   // per 16 tokens: a bad page
    typedef float f16v __attribute__((ext_vector_type(16)));
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
    const int t = lane & 15, g = lane >> 4, col = lane & 31, half = lane >> 5;
    const int nct = P.head->nct;
    const int64_t T1 = P.head->T1, Q = T1 * A.c.nkv, G = min((int64_t)A.grid, (Q + 3) / 4);
    // consecutive parts on one XCD (workgroups go round the 8 of them)
    const int per = (A.grid + 7) / 8, b = (blockIdx.x & 7) * per + (blockIdx.x >> 3);
    if (b >= G) return;
    int64_t u = kv_div((int64_t)b * Q, G);
    const int64_t end = kv_div(((int64_t)b + 1) * Q, G);
    int head = (int)kv_div(u, T1), ct = 0;
    {   // the segment row that holds u
        const int64_t u1 = u - head * T1;
        int lo = 0, hi = nct;
        while (hi - lo > 1) {
            const int step = (hi - lo + 255) / 256, c = lo + tid * step;
            const int k = __syncthreads_count(c < hi && P.up[c] <= u1);
            lo += (k - 1) * step;
            hi = min(hi, lo + step);
        }
        ct = lo;
    }
    for (bool begin = true; u < end && head < A.c.nkv; begin = false) {
        const int64_t qs = head * T1 + P.up[ct] + kExtra;   // its first tile's unit
        Row z = P.row[ct];
        uniform(z);
        const bool shrt = z.nt <= kWhole;   // all of it, or nothing where the cut is inside
        const int i0 = shrt ? 0 : (int)max(u - qs, (int64_t)0), i1 = !shrt ? (int)min((int64_t)z.nt, end - qs) : u > qs - kExtra ? 0 : z.nt;
        if (begin && tid == 0) P.info[b] = Plan::Info{qs, qs + z.nt, ct, head};
        if (i1 > i0 && z.cols > 0) {
        // this lane's column and its q as matrix operands
        const int c = wave * 32 + col;
        const bool ok = c < z.cols;
        const int cc = z.c0 + (ok ? c : 0), row = cc / A.group, pos = ok ? max(z.len - z.n + row, -1) : -1;
        kv_h8 qh[HD / 16], ql[HD / 16];
        float inv, m = -INFINITY, ms = -kBias, l = 0.f;
        f16v o[HD / 32];
#pragma unroll
        for (int d = 0; d < HD / 32; ++d) o[d] = f16v{0.f};
        // what every column of the block sees, what any of them does
        const int posa = z.len - z.n + z.c0 / A.group, posb = z.hi - 1;
        const int vis_all = posa + 1, lo_all = A.window > 0 ? max(0, posb + 1 - A.window) : 0;
        const int lo_any = A.window > 0 ? max(0, max(posa, 0) + 1 - A.window) : 0;
        const int32_t *pages = A.b.pages + (int64_t)z.seq * A.b.max_pages;
        auto edge = [&](int i) KV_INLINE { return z.a + i * TILE + TILE > vis_all || z.a + i * TILE < lo_all; };

        // A wave brings 16 tokens: of k and of v (TT = 2), or waves 0, 1 of k and 2, 3 of v.
        const int part = TT == 2 ? wave : wave & 1;
        const bool mine_k = TT == 2 || wave < 2, mine_v = TT == 2 || wave >= 2;
        KvFrag<DT, HD> kf, vf2;
        KvFrag<DT, HD> &vf = TT == 1 ? kf : vf2;   // (a wave brings one of them)
        int kbad = 0;
        bool odd = false;   // an inf or NaN in v that some rows may not see
        const uint32_t off = KvFrag<DT, HD>::lane_off(t, g), eoff = KvFrag<DT, HD>::lane_eoff(t, g);
        // the first of this wave's 16 rows of tile i
        auto row_of = [&](int i, int *bad) KV_INLINE {
            const int t0 = z.a + i * TILE + 16 * part;
            const int page = z.hi > 0 ? kv_word(pages, min(t0, z.hi - 1) >> A.c.shift) : -1;
            const bool ok = kv_page_ok(A.c, page);
            *bad = !ok && t0 < z.hi && t0 + 16 > lo_any;   // (behind every row's window a page may be anything)
            return kv_slot(A.c, ok ? page : 0, head, t0 & ((1 << A.c.shift) - 1));
        };
        auto fetch_k = [&](int i, KvFrag<DT, HD> &f) KV_INLINE {
            if (!mine_k) return;
            const uint64_t slot = row_of(i, &kbad);
            f.load(A.c.k + slot * R::ROW, A.c.ks + slot * (HD / 32), off, eoff);
        };
        auto fetch_v = [&](int i) KV_INLINE {
            if (!mine_v) return;
            int bad;
            const uint64_t slot = row_of(i, &bad);
            vf.load(A.c.v + slot * R::ROW, A.c.vs + slot * (HD / 32), off, eoff);
        };
        auto store_k = [&](const KvFrag<DT, HD> &f, int n) KV_INLINE {
            if (!mine_k) return;
#pragma unroll
            for (int j = 0; j < R::NL; ++j)
#pragma unroll
                for (int k = 0; k < SPC; ++k)
                    *(kv_h8 *)&kb[n][(16 * part + t) * KROW + 4 * R::CH * j + R::CH * g + 8 * k] = f.eight(j, k);
            if (lane == 0) {
                fbad[n][part] = kbad;
                if (kbad) raise_err(A.err);
            }
        };
        auto store_v = [&](int i, int n) KV_INLINE {
            if (!mine_v) return;
            const bool e = edge(i);
            const int tok = z.a + i * TILE + 16 * part + t;
            if (e && (tok >= z.hi || tok < lo_any)) vf.zero();   // whatever a stale slot holds
#pragma unroll
            for (int j = 0; j < R::NL; ++j)
#pragma unroll
                for (int k = 0; k < SPC; ++k) {
                    const kv_h8 v = vf.eight(j, k);
                    if (e) odd |= kv_odd(v);
                    *(kv_h8 *)&vb[n][(16 * part + t) * VROW + 4 * R::CH * j + R::CH * g + 8 * k] = v;
                }
        };
        kv_h8 ph[2 * TT], pl[2 * TT];
        const float minus = kv_minus();
        // Weights of two scores, pair p of 8 TT (4 pairs make one operand of the values' products): their
        // exponentials, and two pairs later, when those have come, the sum (which would else be put behind the
        // products) and the two terms.
        float e0[3], e1[3];
        auto expo = [&](const f16v(&s)[TT], int p) KV_INLINE {
            const int r = 2 * p % 16;
            e0[p % 3] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[p / 8][r], inv, -ms));
            e1[p % 3] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[p / 8][r + 1], inv, -ms));
        };
        auto finish = [&](int p) KV_INLINE {
            const int k = p / 4, e = 2 * p % 8;
            const float p0 = e0[p % 3], p1 = e1[p % 3];
            l += p0;
            l += p1;
            asm volatile("" : "+v"(l));   // (here)
            kv_h2 hi, lo;
            kv_split2(p0, p1, minus, &hi, &lo);
            ph[k][e] = hi[0];
            ph[k][e + 1] = hi[1];
            pl[k][e] = lo[0];
            pl[k][e + 1] = lo[1];
        };
        auto weigh = [&](const f16v(&s)[TT], int p) KV_INLINE {
            if (p > 1) finish(p - 2);
            expo(s, p);
            if (p == 8 * TT - 1) finish(p - 1), finish(p);
        };
        // The products of a step in pairs (both terms of an operand): NQ of scores (of the k rows in buffer nk into
        // `next`), NV of values (of buffer nv into o) with the weights of `cur`. Operands are read two pairs
        // ahead, and the weights are spread over the pairs before the last operand of weights is due: the order is
        // kept by the barriers, so that products and exponentials run side by side in one wave.
        constexpr int NQ = TT * HD / 16, DV = HD / 32, NV = 2 * TT * DV, NP = 8 * TT;
        static_assert(5 * (NQ + (2 * TT - 1) * DV) / NP < NQ && (TT == 1 || (9 * (NQ + 3 * DV) / NP < NQ + DV && 13 * (NQ + 3 * DV) / NP < NQ + 2 * DV)),
                      "an operand of weights is whole before its products");
        auto products = [&](bool with_scores, int nk, f16v(&next)[TT], int nv, const f16v(&cur)[TT]) KV_INLINE {
            constexpr int AHEAD = 2;
            const int c0 = with_scores ? 0 : NQ, span = NQ + (2 * TT - 1) * DV;
            kv_h8 op[AHEAD + 1];
            auto read = [&](int c) KV_INLINE {
                kv_h8 &w = op[c % (AHEAD + 1)];
                if (c < NQ) {
                    w = *(const kv_h8 *)&kb[nk][(32 * (c / (HD / 16)) + col) * KROW + 16 * (c % (HD / 16)) + 8 * half];
                } else if (c < NQ + NV) {
                    const int k = (c - NQ) / DV, d = (c - NQ) % DV;
                    const _Float16 *p = &vb[nv][(16 * k + 4 * half + (t >> 2)) * VROW + 32 * d + 16 * (g & 1) + (t & 3) * 4];
                    const kv_h4 v0 = kv_tr16(p), v1 = kv_tr16(p + 8 * VROW);
                    w = kv_h8{v0[0], v0[1], v0[2], v0[3], v1[0], v1[1], v1[2], v1[3]};
                }
            };
#pragma unroll
            for (int c = 0; c < AHEAD; ++c) read(c0 + c);
#pragma unroll
            for (int c = 0; c < NQ + NV; ++c) {
                if (c < c0) continue;
                read(c + AHEAD);
                const kv_h8 w = op[c % (AHEAD + 1)];
                if (c < NQ) {
                    const int tt = c / (HD / 16), k = c % (HD / 16);
                    next[tt] = __builtin_amdgcn_mfma_f32_32x32x16_f16(w, ql[k], k ? next[tt] : f16v{0.f}, 0, 0, 0);
                    next[tt] = __builtin_amdgcn_mfma_f32_32x32x16_f16(w, qh[k], next[tt], 0, 0, 0);
                } else {
                    const int k = (c - NQ) / DV, d = (c - NQ) % DV;
                    o[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(w, pl[k], o[d], 0, 0, 0);
                    o[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(w, ph[k], o[d], 0, 0, 0);
                }
#pragma unroll
                for (int p = 0; p < NP; ++p)
                    if (with_scores && p * span / NP == c) weigh(cur, p);
                __builtin_amdgcn_sched_barrier(0);
            }
        };
        auto scores = [&](int n, f16v(&s)[TT]) KV_INLINE {
#pragma unroll
            for (int tt = 0; tt < TT; ++tt) {
                s[tt] = f16v{0.f};
#pragma unroll
                for (int k = 0; k < HD / 16; ++k) {
                    const kv_h8 kk = *(const kv_h8 *)&kb[n][(32 * tt + col) * KROW + 16 * k + 8 * half];
                    s[tt] = __builtin_amdgcn_mfma_f32_32x32x16_f16(kk, ql[k], s[tt], 0, 0, 0);
                    s[tt] = __builtin_amdgcn_mfma_f32_32x32x16_f16(kk, qh[k], s[tt], 0, 0, 0);
                }
            }
        };
        auto largest = [&](const f16v(&s)[TT]) KV_INLINE {
            float x = -INFINITY;
#pragma unroll
            for (int tt = 0; tt < TT; ++tt)
#pragma unroll
                for (int r = 0; r < 16; r += 2) x = fmaxf(fmaxf(x, s[tt][r]), s[tt][r + 1]);
            return x * inv;
        };
        // what the columns do not see of tile i (in buffer n)
        auto mask = [&](int i, int n, f16v(&s)[TT], float &tm) KV_INLINE {
            int badm = 0;
#pragma unroll
            for (int j = 0; j < 2 * TT; ++j) badm |= fbad[n][j] << j;
            badm = __builtin_amdgcn_readfirstlane(badm);
            int passes = __builtin_amdgcn_readfirstlane(edge(i) || badm);
            asm volatile("" : "+s"(passes));   // (a loop of one pass or none: a branch becomes selects, or copies of the scores, in every tile)
            for (; passes; --passes) {
                int last = pos - z.a - i * TILE;
                asm volatile("" : "+v"(last));   // (nor made ahead of the loop)
                const uint32_t w = A.window > 0 ? (uint32_t)A.window : (uint32_t)INT32_MAX;
#pragma unroll
                for (int tt = 0; tt < TT; ++tt)
#pragma unroll
                    for (int r = 0; r < 16; ++r) {   // 0 <= last - k < w
                        const int k = 32 * tt + 8 * (r / 4) + 4 * half + r % 4;
                        const float v = badm >> (2 * tt + r / 8) & 1 ? NAN : s[tt][r];
                        s[tt][r] = (uint32_t)last - (uint32_t)k < w ? v : -INFINITY;
                    }
                tm = largest(s);
            }
        };
        auto raise = [&](float tm) KV_INLINE {
            if (!__ballot(tm > m + kLag)) return;
            const float mn = fmaxf(m, fmaxf(tm, __shfl_xor(tm, 32, 64)));
            const float al = mn == m ? 1.f : __builtin_amdgcn_exp2f(m - mn);
            m = mn;
            ms = mn == -INFINITY ? -kBias : mn - kBias;
            l *= al;
#pragma unroll
            for (int d = 0; d < HD / 32; ++d) o[d] *= al;
        };
        f16v sc[TT], sn[TT];
        {
            KvFrag<DT, HD> k1;
            fetch_k(i0, kf);
            const int b0 = kbad;
            fetch_v(i0);
            fetch_k(i0 + 1, k1);   // (past the last tile: the last page again, never used)
            const int b1 = kbad;
            {
                const float *src = A.q + ((int64_t)(z.r0 + row) * A.nh + head * A.group + cc - row * A.group) * HD + 8 * half;
                float mx = 0.f;
#pragma unroll
                for (int k = 0; k < HD / 16; ++k) {
                    const float4 v0 = *(const float4 *)(src + 16 * k), v1 = *(const float4 *)(src + 16 * k + 4);
                    const float v[8] = {v0.x, v0.y, v0.z, v0.w, v1.x, v1.y, v1.z, v1.w};
#pragma unroll
                    for (int e = 0; e < 8; ++e) mx = fmaxf(mx, fabsf(v[e] * A.qscale));
                }
                mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
                const int ex = min(max((int)(__float_as_uint(mx) >> 23) - 126, -100), 128);
                const float up = __uint_as_float((uint32_t)(13 - ex + 127) << 23);
                inv = __uint_as_float((uint32_t)(ex - 13 + 127) << 23);
#pragma unroll
                for (int k = 0; k < HD / 16; ++k) {
                    const float4 v0 = *(const float4 *)(src + 16 * k), v1 = *(const float4 *)(src + 16 * k + 4);
                    const float v[8] = {v0.x, v0.y, v0.z, v0.w, v1.x, v1.y, v1.z, v1.w};
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        _Float16 hi, lo;
                        kv_split(ok ? v[e] * A.qscale * up : 0.f, &hi, &lo);
                        qh[k][e] = hi;
                        ql[k][e] = lo;
                    }
                }
            }
            kbad = b0;
            store_k(kf, 0);
            kbad = b1;
            store_v(i0, 0);
            store_k(k1, 1);
        }
        __syncthreads();
        if (i0 + 2 < i1) fetch_k(i0 + 2, kf);
        if (i0 + 1 < i1) fetch_v(i0 + 1);
        scores(0, sc);
        {
            float tm = largest(sc);
            mask(i0, 0, sc, tm);
            raise(tm);
        }
        __syncthreads();
        // tile i from its scores to its values, and the scores of tile i + 1
        auto step = [&](int i, int n, f16v(&cur)[TT], f16v(&next)[TT]) KV_INLINE {
            store_k(kf, n);
            store_v(i + 1, 1 - n);
            if (i + 3 < i1) fetch_k(i + 3, kf);
            if (i + 2 < i1) fetch_v(i + 2);
            products(true, 1 - n, next, n, cur);
            float tm = largest(next);
            mask(i + 1, 1 - n, next, tm);
            raise(tm);
            __syncthreads();
        };
        int i = i0;
        for (; i + 2 < i1; i += 2) {
            step(i, 0, sc, sn);
            step(i + 1, 1, sn, sc);
        }
        if (i + 1 < i1) {
            step(i, 0, sc, sn);
#pragma unroll
            for (int tt = 0; tt < TT; ++tt) sc[tt] = sn[tt];
            ++i;
        }
#pragma unroll
        for (int p = 0; p < NP; ++p) weigh(sc, p);
        products(false, 0, sn, (i - i0) & 1, sc);
        if (odd) P.odd[(int64_t)head * nct + ct] = 1, P.head->any = 1;
        __syncthreads();
        l += __shfl_xor(l, 32, 64);
        const bool whole = i0 == 0 && i1 == z.nt;
        if (ok) {
            float *const slot = A.part + (2 * (uint64_t)b + (begin ? 0 : 1)) * F::SLOT;
#pragma unroll
            for (int d = 0; d < HD / 32; ++d)
#pragma unroll
                for (int r = 0; r < 16; r += 4) {
                    const kv_f4 v = {o[d][r], o[d][r + 1], o[d][r + 2], o[d][r + 3]};
                    const int e = 32 * d + 2 * r + 4 * half;
                    if (whole) many_out<HD>(A, z, cc, head, e, v, m, l);
                    else *(kv_f4 *)&slot[c * HD + e] = v;
                }
            if (!whole && half == 0) {
                slot[kCols * HD + 2 * c] = m;
                slot[kCols * HD + 2 * c + 1] = l;
            }
        }
        }
        u = qs + z.nt;
        if (++ct == nct) {
            ct = 0;
            ++head;
        }
    }
}

// One row of one head by itself, token by token: a thread a token for the
// scores, then a thread an element for the weighted sum. Slow, for values that
// a sound model does not have: 4 ms for a row of 16000 tokens. One token with
// an inf in v, of one k/v head or of all: 4000 rows 0.35 ms -> 0.4 to 2.1, 512
// rows behind 16000 tokens 0.3 -> 4.4 and 17.
template <int DT, int HD>
__device__ void lone_row(const KvAttnArgs &A, const Row &q, int col, int head) {
    __shared__ float qs[HD], sc[256], red[4];
    __shared__ uint64_t sl[256];
    const int row = col / A.group, h = head * A.group + col - row * A.group, t = threadIdx.x;
    const int64_t o = ((int64_t)(q.r0 + row) * A.nh + h) * HD;
    const int pos = q.len - q.n + row, lo = A.window > 0 ? max(0, pos + 1 - A.window) : 0;
    auto value = [&](const uint8_t *src, const uint8_t *exps, uint64_t slot, int e) {
        if constexpr (DT == MH_KV_F16) return mh_f16(((const uint16_t *)src)[slot * HD + e]);
        const mh_v2f p = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4((uint32_t)src[(slot * HD + e) / 2],
                                                                  __uint_as_float((uint32_t)exps[slot * (HD / 32) + e / 32] << 23), 0);
        return e & 1 ? p.y : p.x;
    };
    __syncthreads();
    if (t < HD) qs[t] = A.q[o + t] * A.qscale;
    __syncthreads();
    float m = -INFINITY, l = 0.f, acc = 0.f;
    for (int base = lo; base <= pos; base += 256) {
        const int n = min(256, pos + 1 - base);
        float x = -INFINITY;
        if (t < n) {
            const int tok = base + t, page = A.b.pages[(int64_t)q.seq * A.b.max_pages + (tok >> A.c.shift)];
            const bool ok = kv_page_ok(A.c, page);
            const uint64_t slot = kv_slot(A.c, ok ? page : 0, head, tok & ((1 << A.c.shift) - 1));
            sl[t] = slot;
            float d = 0.f;
            for (int e = 0; e < HD; ++e) d = __builtin_fmaf(qs[e], value(A.c.k, A.c.ks, slot, e), d);
            x = ok ? d : NAN;
        }
        const float mx = wave_max(x);
        if ((t & 63) == 0) red[t >> 6] = mx;
        __syncthreads();
        const float mn = fmaxf(m, fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3])));
        const float p = t < n ? __builtin_amdgcn_exp2f(x - mn) : 0.f, al = m == mn ? 1.f : __builtin_amdgcn_exp2f(m - mn);
        sc[t] = p;
        const float ps = wave_sum_dpp(p);
        __syncthreads();
        if ((t & 63) == 0) red[t >> 6] = ps;
        __syncthreads();
        l = l * al + ((red[0] + red[1]) + (red[2] + red[3]));
        m = mn;
        if (t < HD) {
            acc *= al;
            for (int j = 0; j < n; ++j) acc = __builtin_fmaf(sc[j], value(A.c.v, A.c.vs, sl[j], t), acc);
        }
        __syncthreads();
    }
    if (A.sink) l += __builtin_amdgcn_exp2f(A.sink[h] * 1.44269504088896341f - m);
    if (t < HD) A.out[o + t] = pos < 0 ? 0.f : acc / l;
}

// Joins the partial results of the segment that the cut at the beginning of
// block b divides, with the other blocks whose beginning divides it and four
// of each (blockIdx.y). Bound by memory where a prompt's segments lie in two
// parts each (13 us for 67 MB after 4000 tokens). Then the odd segments, row
// by row: where a later token's v is an inf or NaN, its products with weights
// of 0 are not.
template <int DT, int HD>
__global__ void __launch_bounds__(256) k_kv_pjoin(KvAttnArgs A, Plan P) {
    constexpr int SLOT = kCols * (HD + 2);
    __shared__ float sm[256], sl[256];
    __shared__ kv_f4 sv[256];
    const int nct = P.head->nct, b = blockIdx.x + 1, t = threadIdx.x;
    const bool any = P.head->any;
    const int64_t Q = P.head->T1 * A.c.nkv, G = min((int64_t)A.grid, (Q + 3) / 4);
    const Plan::Info I = P.info[b];   // (written where b < G, looked at only there)
    if (b < G) {
        const int64_t at = kv_div((int64_t)b * Q, G);
        const int b0 = (int)kv_div((I.qs + 1) * G - 1, Q), b1 = (int)kv_div(I.qe * G - 1, Q);
        const bool late = kv_div((int64_t)b0 * Q, G) < I.qs - kExtra;   // the first block began in an earlier segment
        if (I.qe - I.qs > kWhole && at > I.qs && !P.odd[(int64_t)I.head * nct + I.ct]) {
            const Row z = P.row[I.ct];
            // Blocks b0 + 1 .. b1 all find this segment: each takes a share of it. 8 partial results a trip to
            // memory; where there are over 16, 8 threads of an element take them in turn (8000 tokens in 63 parts: 8
            // us, one thread 24; 2000 tokens in 13 parts: 12 us, one thread 9).
            const int ks = b1 - b0 < 16 ? 1 : 8, per = 256 / ks, kg = t / per, items = z.cols * (HD / 4);
            for (int i0 = ((b - b0 - 1) * 4 + blockIdx.y) * per; i0 < items; i0 += (b1 - b0) * 4 * per) {
                const int i = min(i0 + t % per, items - 1), c = i / (HD / 4), d = 4 * (i % (HD / 4));
                float M = -INFINITY, L = 0.f;
                kv_f4 v = {0.f, 0.f, 0.f, 0.f};
                auto add = [&](float m, float l, kv_f4 w) KV_INLINE {   // (one that saw nothing has zeros, or NaN)
                    const float g = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - M);
                    v += w * g;
                    L += l * g;
                };
                for (int k0 = b0 + 8 * kg; k0 <= b1; k0 += 8 * ks) {
                    float mk[8], lk[8], mn = M;
                    kv_f4 vk[8];
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        mk[j] = -INFINITY;
                        if (k0 + j <= b1) {
                            const float *s = A.part + (2 * (uint64_t)(k0 + j) + (k0 + j == b0 && late ? 1 : 0)) * SLOT;
                            mk[j] = s[kCols * HD + 2 * c];
                            lk[j] = s[kCols * HD + 2 * c + 1];
                            vk[j] = *(const kv_f4 *)&s[c * HD + d];
                        }
                    }
#pragma unroll
                    for (int j = 0; j < 8; ++j) mn = fmaxf(mn, mk[j]);
                    const float f = M == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(M - mn);
                    v *= f;
                    L *= f;
                    M = mn;
#pragma unroll
                    for (int j = 0; j < 8; ++j)
                        if (k0 + j <= b1) add(mk[j], lk[j], vk[j]);
                }
                if (ks > 1) {
                    sm[t] = M;
                    sl[t] = L;
                    sv[t] = v;
                    __syncthreads();
                    for (int k = 0; k < 8; ++k) M = fmaxf(M, sm[k * 32 + (t & 31)]);
                    v = kv_f4{0.f, 0.f, 0.f, 0.f};
                    L = 0.f;
                    for (int k = 0; k < 8; ++k) add(sm[k * 32 + (t & 31)], sl[k * 32 + (t & 31)], sv[k * 32 + (t & 31)]);
                    __syncthreads();
                }
                if (kg == 0 && i0 + t % per < items) many_out<HD>(A, z, z.c0 + c, I.head, d, v, M, L);
            }
        }
    }
    if (!any) return;
    // (a column a block: a segment's 128 in one block would take it half a second behind 16000 tokens)
    for (int64_t i = (int64_t)blockIdx.x * 4 + blockIdx.y; i < (int64_t)nct * A.c.nkv * kCols; i += (int64_t)gridDim.x * 4) {
        const int64_t seg = i / kCols;
        const int c = (int)(i - seg * kCols);
        if (!P.odd[seg]) continue;
        const Row z = P.row[seg % nct];
        if (c < z.cols) lone_row<DT, HD>(A, z, z.c0 + c, (int)(seg / nct));
    }
}

int many_grid(int hd) { return device_cus() * (hd <= 128 ? 2 : 1); }
constexpr int kGridMax = 2 * 256;

uint64_t up16(uint64_t v) { return (v + 15) / 16 * 16; }

struct Layout {
    uint64_t n_ct, head, row, off, odd, info, part, bytes;
};
Layout layout(const mh_kv_batch &b, int group, int hd, int nkv) {
    const uint64_t n_ct = ((uint64_t)b.n_rows * group + kCols - 1) / kCols + b.n_seqs;
    Layout L;
    L.n_ct = n_ct;
    L.head = up16(8 * (n_ct + 1));
    L.row = L.head + sizeof(Plan::Head);
    L.off = L.row + sizeof(Row) * n_ct;
    L.odd = L.off + up16(4 * ((uint64_t)b.n_seqs + 1));
    L.info = L.odd + up16(4 * n_ct * nkv);
    L.part = L.info + up16(sizeof(Plan::Info) * kGridMax);
    L.bytes = L.part + 2ull * kGridMax * kCols * (hd + 2) * 4;
    return L;
}

template <int DT, int HD>
void many_launch(const KvAttnArgs &A, const Plan &P, int room) {
    MH_LAUNCH("kv_plan", k_kv_plan, dim3(1), dim3(1024), 0, stream(), A, P, KvMany<DT, HD>::TILE, room);
    MH_LAUNCH("kv_many", (k_kv_many<DT, HD>), dim3((unsigned)(A.grid + 7) / 8 * 8), dim3(256), 0, stream(), A, P);
    MH_LAUNCH("kv_pjoin", (k_kv_pjoin<DT, HD>), dim3((unsigned)A.grid - 1, 4), dim3(256), 0, stream(), A, P);
}

template <int DT>
void many_hd(const KvAttnArgs &A, const Plan &P, int room) {
    switch (A.c.hd) {
    case 32: return many_launch<DT, 32>(A, P, room);
    case 64: return many_launch<DT, 64>(A, P, room);
    case 96: return many_launch<DT, 96>(A, P, room);
    case 128: return many_launch<DT, 128>(A, P, room);
    case 192: return many_launch<DT, 192>(A, P, room);
    }
    return many_launch<DT, 256>(A, P, room);
}

}  // namespace

uint64_t kv_many_ws(const mh_kv_cache &c, const mh_kv_batch &b, int group) { return layout(b, group, c.head_dim, c.n_kv_heads).bytes; }

int kv_many_run(const mh_kv_cache &c, const mh_kv_batch &b, KvAttnArgs A, void *ws) {
    const Layout L = layout(b, A.group, c.head_dim, c.n_kv_heads);
    uint8_t *w = (uint8_t *)ws;
    const Plan P{(int64_t *)w, (Row *)(w + L.row), (int32_t *)(w + L.off), (int32_t *)(w + L.odd),
                 (Plan::Head *)(w + L.head), (Plan::Info *)(w + L.info)};
    A.part = (float *)(w + L.part);
    A.grid = std::min(many_grid(c.head_dim), kGridMax);
    if (c.dt == MH_KV_F16) many_hd<MH_KV_F16>(A, P, (int)L.n_ct);
    else many_hd<MH_KV_MXFP4>(A, P, (int)L.n_ct);
    return hip_check(hipGetLastError(), "kv attention launch");
}

}  // namespace mh
