// mh_verify.hip — which drafted tokens the target's probabilities keep, and the
// token after them (mh_verify_dev).
//
// k_vf_part reads every row once: the largest logit and the sum of weights of
// each slice of it. k_vf_walk, a block a sequence, joins the slices, walks down
// the tree and finds the next token in the slice that holds it. Where drafts
// were drawn, a refusal leaves max(p - a q, 0) of a row, whose sum no earlier
// launch has: k_vf_rest adds it up over the whole chip, and the last of a
// sequence's blocks walks on. A chain has one refusal at most, and takes one
// such launch; trees (and chains given by their parents) get kRounds of them,
// and what is refused beyond is added up by a block by itself. 17 rows of 201088:
// 23 us with none refused, of them 1.2 a launch that finds nothing to do; 29, 32
// and 41 with 1, 2 and 4; then 70 to 75 a refusal, 0.9 ms for 16 (8 such
// sequences 1.3 ms).
//
// Why 64 bits: a refusal and the token after it compare a draw with sums over
// the whole vocabulary. Of 201088 normal logits (deviations 0.01 to 4), weights
// of 32 bits in sums of 64 give another token than the definition's for one
// draw in 100000 to one in 4000, sums of 32 bits for one in two to seven. A
// weight costs 20 instructions of 64 bits, each as long as one of 32.
#include <math.h>

#include "mh_kvtree.cuh"

#define VF_INLINE __attribute__((always_inline))

namespace mh {
namespace {

constexpr int kThreads = 256, kWaves = kThreads / 64;   // of a block that reads logits
constexpr int kMaxSlices = 256;                         // of a row
constexpr int kWalk = 512;                              // threads of a block that walks
constexpr int kRounds = 4;
constexpr int kHeld = 2048;                             // slices' sums of a sequence that the walk keeps

// What a slice of a row's logits adds up to, and a whole row's.
struct __attribute__((aligned(16))) Part {
    double z;       // sum of 2^((x - m) heat) (0: no token, NaN: a row without probabilities); temp <= 0: 0 or NaN
    float m;        // largest logit
    int32_t at;     // its first token (temp <= 0)
};

// A row of a tree as the walk sees it (lane i of every wave has row i).
struct __attribute__((aligned(16))) Rows {
    int par, tok;   // par -1: none (or a draft outside the vocabulary)
    float u, x, q;  // its draw, and its logit and its draft's probability in the row that it follows
    int pad[3];
};

// Where a walk stands that waits for the sum of max(p - alpha q, 0) of its row.
struct __attribute__((aligned(16))) Walk {
    double alpha;
    int32_t cur, at, n_kept;   // the row, the last draft that was looked at, kept rows
    int32_t waits;
    unsigned done;             // blocks that have left their sums
    int32_t pad;
};

struct VfArgs {
    const float *x, *q, *u;
    const int32_t *row0, *parent, *token;
    int32_t *n_kept, *kept, *next;
    Part *part;       // [n_rows][slices]
    Part *row;        // [n_rows]
    Rows *info;       // [n_seqs][kTreeRows]
    Walk *walk;       // [n_seqs]
    double *rest;     // [n_seqs][rslices]
    unsigned *err;
    int64_t ld, ldq, V, slice, rslice;
    double heat;      // log2(e) / temp
    int n_seqs, n_rows, max_rows, slices, rslices;
};

enum { GREEDY = 0, CHOSEN = 1, DRAWN = 2 };   // temp <= 0; drafts without probabilities; with

// Lane exchanges of 64 bits without LDS: v of the lane that CTRL names (0
// where it names none or ROWS leaves the row out).
template <int CTRL, int ROWS>
__device__ __forceinline__ double dpp64(double v) {
    const long long b = __double_as_longlong(v);
    const int lo = __builtin_amdgcn_update_dpp(0, (int)b, CTRL, ROWS, 0xF, true), hi = __builtin_amdgcn_update_dpp(0, (int)(b >> 32), CTRL, ROWS, 0xF, true);
    return __longlong_as_double((long long)((uint64_t)(uint32_t)hi << 32 | (uint32_t)lo));
}
__device__ __forceinline__ double lane64(double v, int lane) {   // (the same lane for the wave)
    const long long b = __double_as_longlong(v);
    const int lo = __builtin_amdgcn_readlane((int)b, lane), hi = __builtin_amdgcn_readlane((int)(b >> 32), lane);
    return __longlong_as_double((long long)((uint64_t)(uint32_t)hi << 32 | (uint32_t)lo));
}
// Inclusive sum over the wave's lanes in order; the wave's sum.
__device__ __forceinline__ double wave_scan64(double v) {
    v += dpp64<0x111, 0xF>(v);   // row_shr:1, 2, 4, 8
    v += dpp64<0x112, 0xF>(v);
    v += dpp64<0x114, 0xF>(v);
    v += dpp64<0x118, 0xF>(v);
    v += dpp64<0x142, 0xA>(v);   // row_bcast:15
    v += dpp64<0x143, 0xC>(v);   // row_bcast:31
    return v;
}
__device__ __forceinline__ double wave_sum64(double v) { return lane64(wave_scan64(v), 63); }

// Weight of logit x beside the largest m of its row: 2^((x - m) heat), 0 for
// x = -inf (and where m is -inf: the comparison drops the NaN). 2^f on [-1/2,
// 1/2] by the polynomial that interpolates it in the 11 Chebyshev nodes (off
// by 3.2e-16 of the value at most), the whole exponent from the low bits of y +
// 1.5 * 2^52.
__device__ __forceinline__ double weight(float x, float m, double heat) {
    const double y = fmax(((double)x - (double)m) * heat, -2000.0), magic = 0x1.8p52;
    const double t = y + magic, f = y - (t - magic);
    double p = 0x1.e6063f9b91935p-28;
    p = __builtin_fma(p, f, 0x1.b675bd687d9b8p-24);
    p = __builtin_fma(p, f, 0x1.62bfd477051e0p-20);
    p = __builtin_fma(p, f, 0x1.ffcb540541227p-17);
    p = __builtin_fma(p, f, 0x1.430913096fcb8p-13);
    p = __builtin_fma(p, f, 0x1.5d87fe9d7ab80p-10);
    p = __builtin_fma(p, f, 0x1.3b2ab6fba1de1p-7);
    p = __builtin_fma(p, f, 0x1.c6b08d703ce45p-5);
    p = __builtin_fma(p, f, 0x1.ebfbdff82c598p-3);
    p = __builtin_fma(p, f, 0x1.62e42fefa3a19p-1);
    p = __builtin_fma(p, f, 1.0);
    return __builtin_ldexp(p, (int)(uint32_t)__double_as_longlong(t));
}

// Four floats of a row from token i on (i a multiple of 4; vec: its address is
// one of 16 bytes), `pad` from `stop` on.
__device__ __forceinline__ void load4(const float *x, int64_t i, int64_t stop, bool vec, float pad, float *v) {
    if (vec && i + 4 <= stop) {
        const float4 f = *(const float4 *)(x + i);
        v[0] = f.x, v[1] = f.y, v[2] = f.z, v[3] = f.w;
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = i + j < stop ? x[i + j] : pad;   // (i may be past stop)
    }
}
__device__ __forceinline__ bool aligned16(const void *p) { return (uintptr_t)p % 16 == 0; }

// Of no sequence, where the ranges of rows ascend (row_parts: where they do not).
__device__ __forceinline__ bool padding(const VfArgs &A, int64_t row) { return A.row0 && (row < A.row0[0] || row >= A.row0[A.n_seqs]); }

// A block per slice of a row (blockIdx.y): its largest logit and its sum of
// weights, or its first largest token. E tokens a thread at a time, the next E
// on their way. Bound by memory and the 20 instructions of a weight, which the
// loads do not hide whole: 208 rows of 201088 (167 MB) 44 us = 3.8 TB/s, the
// first largest tokens (temp <= 0) 30 us = 5.7 TB/s; by
// itself in a loop 40, with weights in 32 bits 32, and with slices of their own
// for the waves of a block, whose streams then lie 45 KB apart, 53.
template <bool FIRST, int E>
__global__ void __launch_bounds__(kThreads, 4) k_vf_part(VfArgs A, int first) {
    constexpr int CHUNK = kThreads * E;
    __shared__ double sz[kWaves];
    __shared__ float sm[kWaves];
    __shared__ int sa[kWaves];
    const int t = threadIdx.x, wave = t >> 6;
    const int64_t row = first + blockIdx.y, begin = (int64_t)blockIdx.x * A.slice, stop = min(begin + A.slice, A.V);
    if (padding(A, row)) return;
    const float *x = A.x + row * A.ld;
    const bool vec = aligned16(x);
    float m = -INFINITY, nx[E], v[E];
    double z0 = 0.0, z1 = 0.0;
    bool odd = false;
    int at = INT32_MAX;
    auto load = [&](int64_t c0) VF_INLINE {
        if (vec && c0 + CHUNK <= stop) {   // (all in one block: none waits for another)
#pragma unroll
            for (int j = 0; j < E / 4; ++j) {
                const float4 f = *(const float4 *)(x + c0 + 4 * (j * kThreads + t));
                nx[4 * j] = f.x, nx[4 * j + 1] = f.y, nx[4 * j + 2] = f.z, nx[4 * j + 3] = f.w;
            }
        } else {
#pragma unroll
            for (int j = 0; j < E; ++j) {
                const int64_t i = c0 + 4 * (j / 4 * kThreads + t) + j % 4;
                nx[j] = x[min(i, stop - 1)];
                nx[j] = i < stop ? nx[j] : -INFINITY;
            }
        }
    };
    load(begin);
    for (int64_t c0 = begin; c0 < stop; c0 += CHUNK) {
#pragma unroll
        for (int j = 0; j < E; ++j) v[j] = nx[j];
        if (c0 + CHUNK < stop) load(c0 + CHUNK);
        float tm = -INFINITY;
#pragma unroll
        for (int j = 0; j < E; ++j) {
            tm = fmaxf(tm, v[j]);
            odd |= FIRST ? v[j] != v[j] : !(v[j] < INFINITY);
        }
        if (tm > m) {
            if (FIRST) {
#pragma unroll
                for (int j = E - 1; j >= 0; --j) at = v[j] == tm ? (int)c0 + 4 * (j / 4 * kThreads + t) + j % 4 : at;
            } else {
                const double w = weight(m, tm, A.heat);
                z0 *= w;
                z1 *= w;
            }
            m = tm;
        }
        if (!FIRST)
#pragma unroll
            for (int j = 0; j < E; j += 2) {
                z0 += weight(v[j], m, A.heat);
                z1 += weight(v[j + 1], m, A.heat);
            }
    }
    const float M = wave_max(m);
    double z = 0.0;
    if (FIRST) at = wave_min(m == M && M != -INFINITY ? at : INT32_MAX);
    else z = wave_sum64((z0 + z1) * weight(m, M, A.heat));
    if (__ballot(odd)) z = NAN;
    if ((t & 63) == 0) sz[wave] = z, sm[wave] = M, sa[wave] = at;
    __syncthreads();
    if (t) return;
    Part p{0.0, sm[0], sa[0]};
    for (int w = 1; w < kWaves; ++w)
        if (sm[w] > p.m || (sm[w] == p.m && sa[w] < p.at)) p.m = sm[w], p.at = sa[w];
    for (int w = 0; w < kWaves; ++w) p.z += FIRST ? sz[w] : sz[w] * weight(sm[w], p.m, A.heat);
    A.part[row * A.slices + blockIdx.x] = p;
}

// The slices of a row that was taken for padding and is a sequence's all the
// same, by one wave. (Looked for among the ranges by the blocks of all padding
// instead, 300 rows of it cost the call 3 us.)
template <bool FIRST>
__device__ __forceinline__ void row_parts(const VfArgs &A, int64_t row) {
    const int lane = threadIdx.x & 63;
    const float *x = A.x + row * A.ld;
    for (int s = 0; s < A.slices; ++s) {
        const int64_t begin = s * A.slice, stop = min(begin + A.slice, A.V);
        float m = -INFINITY;
        double z = 0.0;
        bool odd = false;
        int at = INT32_MAX;
        for (int64_t i = begin + lane; i < stop; i += 64) {
            const float v = x[i];
            odd |= FIRST ? v != v : !(v < INFINITY);
            if (v > m) m = v, at = (int)i;
        }
        const float M = wave_max(m);
        at = wave_min(m == M ? at : INT32_MAX);
        if (!FIRST)
            for (int64_t i = begin + lane; i < stop; i += 64) z += weight(x[i], M, A.heat);
        z = wave_sum64(z);
        if (__ballot(odd)) z = NAN;
        if (lane == 0) A.part[row * A.slices + s] = Part{z, M, at};
    }
    __threadfence();   // (the wave's other lanes read them)
}

// The first of a block's threads at which the running sum of v passes `want`
// (and v > 0; if rounding leaves none, the last with v > 0; -1: none has), and
// the sum before it: the same for all threads.
template <int THREADS>
__device__ __forceinline__ int find(double v, double want, double *before) {
    constexpr int W = THREADS / 64;
    __shared__ double sum[W], past_at[W], last_at[W];
    __shared__ int past_i[W], last_i[W];
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
    const double run = wave_scan64(v);
    __syncthreads();
    if (lane == 63) sum[wave] = run;
    __syncthreads();
    double base = 0.0;
    for (int w = 0; w < wave; ++w) base += sum[w];
    const uint64_t past = __ballot(v > 0.0 && base + run > want), any = __ballot(v > 0.0);
    const int p = past ? __builtin_ctzll(past) : 0, l = any ? 63 - __builtin_clzll(any) : 0;
    const double pb = base + lane64(run - v, p), lb = base + lane64(run - v, l);
    if (lane == 0) {
        past_i[wave] = past ? wave * 64 + p : -1;
        last_i[wave] = any ? wave * 64 + l : -1;
        past_at[wave] = pb;
        last_at[wave] = lb;
    }
    __syncthreads();
    int r = -1, last = -1;
    double rb = 0.0, lastb = 0.0;
    for (int w = 0; w < W; ++w) {
        if (r < 0 && past_i[w] >= 0) r = past_i[w], rb = past_at[w];
        if (last_i[w] >= 0) last = last_i[w], lastb = last_at[w];
    }
    *before = r < 0 ? lastb : rb;
    return r < 0 ? last : r;
}
template <int THREADS>
__device__ __forceinline__ double block_sum64(double v) {
    __shared__ double sum[THREADS / 64];
    v = wave_sum64(v);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) sum[threadIdx.x >> 6] = v;
    __syncthreads();
    double s = 0.0;
    for (int w = 0; w < THREADS / 64; ++w) s += sum[w];
    return s;
}

// What is left of a row's probabilities: weights without the tokens of `gone`,
// or max(w inv - alpha q, 0).
struct Left {
    const float *x, *q;   // q NULL: not drawn, or nothing refused
    double heat, inv, alpha;
    const int *gone;
    float m;
    int n_gone;
    bool xv, qv;

    __device__ __forceinline__ void of(const float *a, const float *b, int64_t i, double *r) const {
        if (q) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const double d = __builtin_fma(-alpha, (double)b[j], weight(a[j], m, heat) * inv);
                r[j] = d > 0.0 ? d : 0.0;   // (a NaN too)
            }
            return;
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) r[j] = weight(a[j], m, heat);
        for (int k = 0; k < n_gone; ++k)
#pragma unroll
            for (int j = 0; j < 4; ++j) r[j] = gone[k] == i + j ? 0.0 : r[j];
    }
    // tokens i .. i + 3 (i a multiple of 4), 0 from `stop` on
    __device__ __forceinline__ void four(int64_t i, int64_t stop, double *r) const {
        float a[4], b[4] = {};
        load4(x, i, stop, xv, -INFINITY, a);
        if (q) load4(q, i, stop, qv, INFINITY, b);
        of(a, b, i, r);
    }
    // the sum over [from, to), `lanes` threads together, this one the lane-th (from a multiple of 4): four loads of
    // each row on their way, those past the end of the last tokens once more
    __device__ __forceinline__ double sum(int64_t from, int64_t to, int lane, int lanes) const {
        constexpr int AT = 4;
        const bool vec = xv && (!q || qv);
        const int n = (int)(to - from), fours = vec ? n / 4 : 0;   // (a slice: less than 2^31)
        double v = 0.0;
        for (int g0 = lane; g0 < fours; g0 += AT * lanes) {
            float4 a[AT], b[AT];
#pragma unroll
            for (int k = 0; k < AT; ++k) a[k] = *(const float4 *)(x + from + 4 * (int64_t)min(g0 + k * lanes, fours - 1));
            if (q)
#pragma unroll
                for (int k = 0; k < AT; ++k) b[k] = *(const float4 *)(q + from + 4 * (int64_t)min(g0 + k * lanes, fours - 1));
#pragma unroll
            for (int k = 0; k < AT; ++k) {
                const float av[4] = {a[k].x, a[k].y, a[k].z, a[k].w}, bv[4] = {b[k].x, b[k].y, b[k].z, b[k].w};
                double r[4];
                of(av, bv, from + 4 * (int64_t)(g0 + k * lanes), r);
                v += g0 + k * lanes < fours ? (r[0] + r[1]) + (r[2] + r[3]) : 0.0;
            }
        }
        for (int64_t i = from + 4 * (int64_t)(fours + lane); i < to; i += 4 * lanes) {
            double r[4];
            four(i, to, r);
            v += (r[0] + r[1]) + (r[2] + r[3]);
        }
        return v;
    }
};

// The first token of [a, b) at which the running sum of what is left passes
// `want`, written to `out`: the part of it that one wave adds up first, until
// every thread can hold four tokens.
template <int THREADS>
__device__ __forceinline__ void pick(const Left &L, int64_t a, int64_t b, double want, int32_t *out) {
    constexpr int W = THREADS / 64;
    __shared__ double part[W];
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
    while (b - a > 4 * THREADS) {
        const int64_t len = ((b - a + W - 1) / W + 3) / 4 * 4, from = min(a + wave * len, b);
        const double v = wave_sum64(L.sum(from, min(from + len, b), lane, 64));
        __syncthreads();
        if (lane == 0) part[wave] = v;
        __syncthreads();
        int at = 0;
        double run = 0.0, before = 0.0;
        for (int w = 0; w < W; ++w) {
            const double p = part[w];
            if (p > 0.0) at = w, before = run;
            run += p;
            if (p > 0.0 && run > want) break;
        }
        want -= before;
        a += at * len;
        b = min(a + len, b);
    }
    double r[4], before;
    L.four(a + 4 * t, b, r);
    const int hit = max(find<THREADS>((r[0] + r[1]) + (r[2] + r[3]), want, &before), 0);
    if (t != hit) return;
    int at = 0;
    double run = before;
    bool found = false;
#pragma unroll
    for (int j = 0; j < 4; ++j) {   // the first past it, or the last with any
        run += r[j];
        if (r[j] > 0.0 && !found) at = j;
        found |= r[j] > 0.0 && run > want;
    }
    *out = (int32_t)min(a + 4 * t + at, b - 1);
}

template <int MODE>
__device__ __forceinline__ Rows rows_of(const VfArgs &A, int r0, int n) {
    const int lane = threadIdx.x & 63;
    Rows R{-1, -1, 0.f, -INFINITY, 0.f, {}};
    if (lane < n) {
        R.par = A.parent ? A.parent[r0 + lane] : lane - 1;
        R.tok = A.token[r0 + lane];
        R.u = A.u[r0 + lane];
        if (R.par < -1 || R.par >= lane) {
            raise_err(A.err);
            R.par = -1;
        }
        if (R.par >= 0 && R.tok >= 0 && R.tok < A.V) {
            if (MODE != GREEDY) R.x = A.x[(int64_t)(r0 + R.par) * A.ld + R.tok];
            if (MODE == DRAWN) R.q = A.q[(int64_t)(r0 + R.par) * A.ldq + R.tok];
        } else {
            R.par = -1;
        }
    }
    return R;
}

// From row `cur` on (with the sums of max(p - alpha q, 0) of its slices in
// `rest` where alpha > 0, and their sum `left`): the drafts that follow it, in
// order, as the bits of a ballot. At the end the slices of the last row, without
// what refused drafts took of them, tell the one in which the running sum
// passes the draw. rows: the sequence's rows; sums: their slices' sums, or NULL
// (both LDS).
template <int MODE, int THREADS>
__device__ __forceinline__ void descend(const VfArgs &A, int s, int r0, const Rows &R, const Part *rows, const double *sums, int cur, int at, int n_kept, double alpha,
                                        double left, const double *rest, bool wait) {
    __shared__ int gone[kTreeRows], in[kTreeRows];   // refused tokens, their slices
    __shared__ double took[kTreeRows], share[kMaxSlices];
    __shared__ int again[kMaxSlices];
    constexpr int W = THREADS / 64;
    __shared__ double part[kTreeRows][W];
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
    int32_t *const kept = A.kept + (int64_t)s * A.max_rows;
    const double w = MODE != GREEDY && R.par >= 0 ? weight(R.x, rows[R.par].m, A.heat) : 0.0;
    uint64_t out = 0;        // the refused drafts after the current row
    double off = 0.0;        // what they took (CHOSEN)
    auto row_left = [&]() VF_INLINE {
        Left L;
        L.x = A.x + (int64_t)(r0 + cur) * A.ld;
        L.q = MODE == DRAWN && alpha > 0.0 ? A.q + (int64_t)(r0 + cur) * A.ldq : nullptr;
        L.heat = A.heat;
        L.inv = 1.0 / rows[cur].z;
        L.alpha = alpha;
        L.gone = gone;
        L.m = rows[cur].m;
        L.n_gone = 0;
        L.xv = aligned16(L.x);
        L.qv = aligned16(L.q);
        return L;
    };
    for (;;) {
        const uint64_t after = __ballot(R.par == cur) & ~((2ull << at) - 1);   // (2 << 63: 0, none after)
        if (!after) break;
        const int i = __builtin_amdgcn_readfirstlane(__builtin_ctzll(after)), c = __builtin_amdgcn_readlane(R.tok, i);
        const double z = rows[cur].z, wc = lane64(w, i), u = (double)__shfl(R.u, i, 64);
        bool yes;
        if (MODE == GREEDY) {
            yes = c == rows[cur].at;
        } else if (MODE == CHOSEN) {
            const bool twice = __ballot((out >> lane & 1) && R.tok == c) != 0;
            at = i;
            if (twice) continue;
            yes = u * (z - off) < wc;
            off += wc;
        } else {
            const double qc = (double)__shfl(R.q, i, 64), d = __builtin_fma(-alpha, qc, wc / z);
            yes = u * qc * left < (d > 0.0 ? d : 0.0);
        }
        at = i;
        if (yes) {
            if (t == 0) kept[n_kept] = i;
            ++n_kept;
            cur = i;
            out = 0;
            off = alpha = 0.0;
            left = 1.0;
            continue;
        }
        out |= 1ull << i;
        if (MODE != DRAWN) continue;
        alpha += left;
        if (wait) {   // for another launch's sum
            if (t == 0) {
                Walk &W = A.walk[s];
                W.alpha = alpha;
                W.cur = cur;
                W.at = at;
                W.n_kept = n_kept;
                W.waits = rows[cur].z > 0.0;
            }
            if (rows[cur].z > 0.0) return;
            break;
        }
        const Left L = row_left();
        left = 0.0;
        __syncthreads();
        for (int k = 0; k < A.rslices; ++k) {
            const double f = block_sum64<THREADS>(L.sum(k * A.rslice, min((k + 1) * A.rslice, A.V), t, THREADS));
            if (t == 0) share[k] = f;
            left += f;
        }
        rest = share;
        __syncthreads();
    }
    if (t == 0) A.n_kept[s] = n_kept;
    if (t >= n_kept && t < A.max_rows) kept[t] = -1;
    if (MODE == GREEDY || !(rows[cur].z > 0.0)) {   // (NaN too)
        if (t == 0) A.next[s] = MODE == GREEDY ? rows[cur].at : -1;
        return;
    }
    const double u0 = (double)__shfl(R.u, 0, 64);
    Left L = row_left();
    if (MODE == DRAWN && alpha > 0.0) {
        const double v = t < A.rslices ? rest[t] : 0.0, sum = block_sum64<THREADS>(v);
        if (sum > 0.0) {
            double before;
            const int sl = max(find<THREADS>(v, u0 * sum, &before), 0);
            pick<THREADS>(L, sl * A.rslice, min((sl + 1) * A.rslice, A.V), u0 * sum - before, A.next + s);
            return;
        }
        L.q = nullptr;   // rounding left nothing: the row's own probabilities
        out = 0;
    }
    // the row's slices without the refused tokens
    if (MODE == CHOSEN && out) {
        L.n_gone = __popcll(out);
        if (wave == 0 && (out >> lane & 1)) {
            const int k = __popcll(out & ((1ull << lane) - 1));
            gone[k] = R.tok;
            in[k] = (int)((uint32_t)R.tok / (uint32_t)A.slice);
            took[k] = w;
        }
    }
    __syncthreads();
    for (int pass = 0; pass < 2; ++pass) {   // (the second: rounding left nothing, the row's own probabilities)
        if (t < kMaxSlices) {
            double all = 0.0;
            if (sums) {
                all = t < A.slices ? sums[cur * A.slices + t] : 0.0;
            } else if (t < A.slices) {
                const Part p = A.part[(int64_t)(r0 + cur) * A.slices + t];
                all = p.z * weight(p.m, L.m, A.heat);
            }
            double less = all;
            for (int k = 0; k < L.n_gone; ++k) less -= in[k] == t ? took[k] : 0.0;
            share[t] = less;
            again[t] = less < all * 0x1p-10;   // (too little of it to be a difference: added up again)
        }
        __syncthreads();
        // (parts of 1024 tokens, or eighths, a wave each; two tokens of a slice find the same)
        const int parts = (int)min(A.slice / 1024, (int64_t)W);
        for (int p = wave; p < L.n_gone * parts; p += W) {
            const int k = p / parts, sl = in[k];
            if (!again[sl]) continue;
            const int64_t len = A.slice / parts, a = sl * A.slice + (p - k * parts) * len, b = min((sl + 1) * A.slice, A.V);
            const double f = a < b ? wave_sum64(L.sum(a, p - k * parts == parts - 1 ? b : min(a + len, b), lane, 64)) : 0.0;
            if (lane == 0) part[k][p - k * parts] = f;
        }
        __syncthreads();
        if (t < L.n_gone && again[in[t]]) {
            double f = 0.0;
            for (int w = 0; w < parts; ++w) f += part[t][w];
            share[in[t]] = f;
        }
        __syncthreads();
        const double v = t < kMaxSlices ? share[t] : 0.0, sum = block_sum64<THREADS>(v);
        if (sum > 0.0) {
            double before;
            const int sl = find<THREADS>(v, u0 * sum, &before);
            pick<THREADS>(L, sl * A.slice, min((sl + 1) * A.slice, A.V), u0 * sum - before, A.next + s);
            return;
        }
        L.n_gone = 0;
        __syncthreads();
    }
    if (t == 0) A.next[s] = -1;
}

// A block per sequence: the rows' sums joined, a wave a row, and the walk.
template <int MODE>
__global__ void __launch_bounds__(kWalk) k_vf_walk(VfArgs A) {
    __shared__ Part rows[kTreeRows];
    __shared__ double sums[kHeld];
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6, s = blockIdx.x;
    const int r0 = A.row0 ? A.row0[s] : s, r1 = A.row0 ? A.row0[s + 1] : s + 1, n = r1 - r0;
    const bool ok = r0 >= 0 && r1 >= r0 && r1 <= A.n_rows && n <= A.max_rows;
    const bool unread = A.row0 && (r0 < A.row0[0] || r1 > A.row0[A.n_seqs]);   // some of its rows were padding to k_vf_part
    if (!ok && t == 0) raise_err(A.err);
    if (MODE == DRAWN && t == 0) A.walk[s].waits = 0, A.walk[s].done = 0;
    int32_t *const kept = A.kept + (int64_t)s * A.max_rows;
    if (!ok || n == 0) {
        if (t < A.max_rows) kept[t] = -1;
        if (t == 0) A.n_kept[s] = 0, A.next[s] = -1;
        return;
    }
    const Rows R = rows_of<MODE>(A, r0, n);
    if (__builtin_expect(unread, false))
        for (int r = wave; r < n; r += kWalk / 64)
            if (padding(A, r0 + r)) row_parts<MODE == GREEDY>(A, r0 + r);
    if (MODE == DRAWN && t < n) A.info[(int64_t)s * kTreeRows + t] = R;
    const bool held = MODE != GREEDY && n * A.slices <= kHeld;
    for (int r = wave; r < n; r += kWalk / 64) {
        const Part *part = A.part + (int64_t)(r0 + r) * A.slices;
        Part p[kMaxSlices / 64];
        float m = -INFINITY;
#pragma unroll
        for (int k = 0; k < kMaxSlices / 64; ++k) {
            const int i = lane + 64 * k;
            p[k] = Part{0.0, -INFINITY, INT32_MAX};
            if (i < A.slices) p[k] = part[i];
            m = fmaxf(m, p[k].m);
        }
        const float M = wave_max(m);
        double z = 0.0;
        int at = INT32_MAX;
#pragma unroll
        for (int k = 0; k < kMaxSlices / 64; ++k) {
            if (MODE == GREEDY) {
                z += p[k].z;
                if (p[k].m == M) at = min(at, p[k].at);
            } else if (k == 0 || A.slices > 64 * k) {
                const double w = p[k].z * weight(p[k].m, M, A.heat);
                z += w;
                if (held && lane + 64 * k < A.slices) sums[r * A.slices + lane + 64 * k] = w;
            }
        }
        z = wave_sum64(z);
        if (MODE == GREEDY) at = wave_min(at);
        if (lane == 0) {
            rows[r] = Part{z, M, z != z || M == -INFINITY ? -1 : at};
            if (MODE == DRAWN) A.row[r0 + r] = rows[r];
        }
    }
    if (t == 0) kept[0] = 0;
    __syncthreads();
    descend<MODE, kWalk>(A, s, r0, R, rows, held ? sums : nullptr, 0, 0, 1, 0.0, 1.0, nullptr, true);
}

// A block per slice of the row at which a sequence (blockIdx.y) waits: its sum
// of max(p - alpha q, 0). The block that finishes last walks on (the counter
// only tells which that is; sums are added in the slices' order).
__global__ void __launch_bounds__(kThreads) k_vf_rest(VfArgs A, int first, int last_round) {
    __shared__ Part rows[kTreeRows];
    __shared__ double rest[kThreads];
    __shared__ bool final;
    const int s = first + blockIdx.y, t = threadIdx.x;
    const Walk W = A.walk[s];
    if (!W.waits) return;
    const int r0 = A.row0 ? A.row0[s] : s, n = (A.row0 ? A.row0[s + 1] : s + 1) - r0;
    const Part p = A.row[r0 + W.cur];
    Left L;
    L.x = A.x + (int64_t)(r0 + W.cur) * A.ld;
    L.q = A.q + (int64_t)(r0 + W.cur) * A.ldq;
    L.heat = A.heat;
    L.inv = 1.0 / p.z;
    L.alpha = W.alpha;
    L.gone = nullptr;
    L.m = p.m;
    L.n_gone = 0;
    L.xv = aligned16(L.x);
    L.qv = aligned16(L.q);
    double *const sums = A.rest + (int64_t)s * A.rslices;
    const int64_t begin = (int64_t)blockIdx.x * A.rslice;
    const double mine = block_sum64<kThreads>(L.sum(begin, min(begin + A.rslice, A.V), t, kThreads));
    if (t == 0) {
        // (the sum is a device-scope store, complete before the count: no cache has to be written back for it)
        __hip_atomic_store(sums + blockIdx.x, mine, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        final = __hip_atomic_fetch_add(&A.walk[s].done, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == (unsigned)A.rslices - 1;
    }
    __syncthreads();
    if (!final) return;
    const int lane = t & 63;
    Rows R{-1, -1, 0.f, -INFINITY, 0.f, {}};
    if (lane < n) R = A.info[(int64_t)s * kTreeRows + lane];
    if (t < n) rows[t] = A.row[r0 + t];
    rest[t] = t < A.rslices ? __hip_atomic_load(sums + t, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) : 0.0;
    if (t == 0) A.walk[s].waits = 0, A.walk[s].done = 0;
    __syncthreads();
    const double left = block_sum64<kThreads>(rest[t]);
    descend<DRAWN, kThreads>(A, s, r0, R, rows, nullptr, W.cur, W.at, W.n_kept, W.alpha, left, rest, !last_round);
}

// How n rows are cut (into at most 256 slices of a row): chunks of 4 tokens a
// thread, one or two of them a block, until chunks of 16 keep all CUs busy. A
// whole call in us, slices of 1024 / 2048 / 4096 / 8192 tokens: 1 row of 201088
// 10.2 / 10.8 / 13.1 / 13.5, 8 rows 15.3 / 15.0 / 16.9 / 16.7, 52 rows 29.8 /
// 26.7 / 26.8 / 28.3, 208 rows 80.5 / 70.9 / 60.6 / 59.4. Measured at that
// vocabulary and temp > 0 only: others, and calls that make no weights, take the
// same cuts by their numbers of logits.
struct Cut {
    int E, slices;
    int64_t slice;
};
Cut cut(int n, int64_t V) {
    const int64_t all = n * V;
    const int E = all < ((int64_t)1 << 23) ? 4 : 16, chunks = all < ((int64_t)1 << 20) || (E == 16 && all < ((int64_t)1 << 25)) ? 1 : 2;
    const int64_t chunk = kThreads * E, most = (V + kMaxSlices - 1) / kMaxSlices;
    const int64_t slice = std::max(chunks * chunk, (most + chunk - 1) / chunk * chunk);
    return Cut{E, (int)((V + slice - 1) / slice), slice};
}
// The last rows of n sequences: at most 64 blocks each, which count at one
// word.
Cut cut_rest(int n, int64_t V) {
    const int64_t most = std::min(64, std::max(1, 512 / n)), per = (V + most - 1) / most, slice = (per + 4095) / 4096 * 4096;
    return Cut{4, (int)((V + slice - 1) / slice), slice};
}

uint64_t part_bytes(uint64_t n_rows, int64_t V) { return std::max<uint64_t>(n_rows, 1) * ((std::min<int64_t>(kMaxSlices, (V + 1023) / 1024) + 1) * sizeof(Part)); }
uint64_t ws_bytes_for(uint64_t n_seqs, uint64_t n_rows, int64_t V) { return part_bytes(n_rows, V) + n_seqs * (sizeof(Walk) + kTreeRows * sizeof(Rows) + 8 * 64); }

template <bool FIRST, int E>
void launch_part(const VfArgs &A, dim3 grid, int first) {
    MH_LAUNCH("verify_part", (k_vf_part<FIRST, E>), grid, dim3(kThreads), 0, stream(), A, first);
}

int validate(int n_seqs, int n_rows, int64_t V, const char *what) {
    if (n_seqs < 1 || n_seqs > (1 << 20) || n_rows < 0 || n_rows >= (1 << 24)) return fail(MH_E_ARG, "%s: %d sequences, %d rows", what, n_seqs, n_rows);
    if (V < 1 || V > (1 << 30)) return fail(MH_E_ARG, "%s: vocabulary of %lld tokens", what, (long long)V);
    return MH_OK;
}

}  // namespace
}  // namespace mh

using namespace mh;

extern "C" {

int mh_verify_ws(int n_seqs, int n_rows, int64_t V, uint64_t *bytes) {
    clear_error();
    MH_TRY(validate(n_seqs, n_rows, V, "mh_verify_ws"));
    if (!bytes) return fail(MH_E_ARG, "mh_verify_ws: NULL result");
    *bytes = ws_bytes_for(n_seqs, n_rows, V);
    return MH_OK;
}

int mh_verify_dev(const mh_draft *d, int32_t *n_kept, int32_t *kept, int32_t *next, void *ws, uint64_t ws_bytes) {
    const char *what = "mh_verify_dev";
    clear_error();
    if (!d) return fail(MH_E_ARG, "%s: NULL drafts", what);
    MH_TRY(validate(d->n_seqs, d->n_rows, d->vocab, what));
    if (d->max_rows < 1) return fail(MH_E_ARG, "%s: max_rows %d", what, d->max_rows);
    if (d->max_rows > kTreeRows) return fail(MH_E_UNSUPPORTED, "%s: trees of %d rows (at most %d)", what, d->max_rows, kTreeRows);
    if (!d->row0 && d->n_rows != d->n_seqs)
        return fail(MH_E_ARG, "%s: without row0 a sequence has one row (%d rows, %d sequences)", what, d->n_rows, d->n_seqs);
    if (!d->logits || !d->token || !d->u || !n_kept || !kept || !next || !ws) return fail(MH_E_ARG, "%s: NULL argument", what);
    const bool greedy = !(d->temp > 0.f), q = d->q && !greedy;
    if (d->temp != d->temp || d->temp > 3e38f || (!greedy && !std::isfinite(1.0 / (double)d->temp))) return fail(MH_E_ARG, "%s: temp %g", what, (double)d->temp);
    const int64_t far = (int64_t)1 << 40;
    if (d->ld < d->vocab || d->ld > far || (d->q && (d->ldq < d->vocab || d->ldq > far)))
        return fail(MH_E_ARG, "%s: rows of %lld and %lld floats, %lld tokens", what, (long long)d->ld, (long long)d->ldq, (long long)d->vocab);
    const uint64_t n = (uint64_t)d->n_rows, ns = (uint64_t)d->n_seqs, need = ws_bytes_for(ns, n, d->vocab);
    if (ws_bytes < need) return fail(MH_E_ARG, "%s: a workspace of %llu bytes, %llu needed", what, (unsigned long long)ws_bytes, (unsigned long long)need);
    if (((uintptr_t)d->logits | (uintptr_t)d->q | (uintptr_t)d->token | (uintptr_t)d->u | (uintptr_t)d->row0 | (uintptr_t)d->parent | (uintptr_t)n_kept |
         (uintptr_t)kept | (uintptr_t)next) % 4 || (uintptr_t)ws % 16)
        return fail(MH_E_ARG, "%s: misaligned argument", what);
    uint64_t xb, qb = 0;
    MH_TRY(rows_bytes(n, d->ld, d->vocab, &xb, what));
    if (d->q) MH_TRY(rows_bytes(n, d->ldq, d->vocab, &qb, what));
    const struct {
        const void *p;
        uint64_t n;
    } mem[] = {{ws, need}, {n_kept, 4 * ns}, {kept, 4 * ns * d->max_rows}, {next, 4 * ns},
               {d->logits, xb}, {d->q, qb}, {d->token, 4 * n}, {d->u, 4 * n}, {d->row0, d->row0 ? 4 * (ns + 1) : 0}, {d->parent, d->parent ? 4 * n : 0}};
    for (int i = 0; i < 4; ++i)   // (what is written, against all)
        for (int j = i + 1; j < 10; ++j)
            if (mem[j].p && kv_overlap(mem[i].p, mem[i].n, mem[j].p, mem[j].n)) return fail(MH_E_ARG, "%s: %p overlaps %p", what, mem[i].p, mem[j].p);
    MH_TRY(require_init());
    OnDevice here;
    for (const auto &r : mem)
        if (r.p && r.n) MH_TRY(resolve_here(r.p, r.n, what));
    unsigned *flag;
    MH_TRY(verify_flag(&flag));
    const Cut c = cut(d->n_rows, d->vocab), r = cut_rest(d->n_seqs, d->vocab);
    Part *const part = (Part *)ws;
    Walk *const walk = (Walk *)((uint8_t *)ws + part_bytes(n, d->vocab));
    Rows *const info = (Rows *)(walk + ns);   // (of each sequence's own: two may name one row, from other places)
    const VfArgs A{d->logits, q ? d->q : nullptr, d->u, d->row0, d->parent, d->token, n_kept, kept, next, part, part + n * c.slices, info, walk,
                   (double *)(info + ns * kTreeRows), flag, d->ld, d->ldq, d->vocab, c.slice, r.slice, greedy ? 0.0 : 1.4426950408889634 / (double)d->temp,
                   d->n_seqs, d->n_rows, d->max_rows, c.slices, r.slices};
    for (int row = 0; row < d->n_rows; row += 32768) {   // (a grid's second axis ends at 65535)
        const dim3 grid((unsigned)c.slices, (unsigned)std::min(32768, d->n_rows - row));
        if (greedy) c.E == 4 ? launch_part<true, 4>(A, grid, row) : launch_part<true, 16>(A, grid, row);
        else c.E == 4 ? launch_part<false, 4>(A, grid, row) : launch_part<false, 16>(A, grid, row);
    }
    const dim3 seqs((unsigned)d->n_seqs);
    if (greedy) MH_LAUNCH("verify_walk", k_vf_walk<GREEDY>, seqs, dim3(kWalk), 0, stream(), A);
    else if (!q) MH_LAUNCH("verify_walk", k_vf_walk<CHOSEN>, seqs, dim3(kWalk), 0, stream(), A);
    else MH_LAUNCH("verify_walk", k_vf_walk<DRAWN>, seqs, dim3(kWalk), 0, stream(), A);
    const int rounds = !q ? 0 : std::min(d->max_rows - 1, d->parent ? kRounds : 1);   // (a chain ends with its first refusal)
    for (int k = 0; k < rounds; ++k)
        for (int s = 0; s < d->n_seqs; s += 32768)
            MH_LAUNCH("verify_rest", k_vf_rest, dim3((unsigned)r.slices, (unsigned)std::min(32768, d->n_seqs - s)), dim3(kThreads), 0, stream(), A, s,
                      (int)(k == rounds - 1));
    return hip_check(hipGetLastError(), "verify launch");
}

}  // extern "C"
