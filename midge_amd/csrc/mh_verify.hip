// mh_verify.hip — which drafted tokens the target's probabilities keep, and the
// token after them (mh_verify_dev).
//
// Two launches read every row once (k_vf_part: the largest logit and the sum of
// weights of each slice of a row) and walk down each tree (k_vf_walk); drafts
// that were drawn take a third where a sequence ends with a refusal
// (k_vf_rest: what max(p - a q, 0) leaves of its last row, which no sum of the
// first launch tells).
//
// Why 64 bits: a refusal and the token after it compare a draw with sums over
// the whole vocabulary. With weights in 32 bits every one of 200000 borders
// between tokens is off by about 2^-24 of the sum, and a draw in some hundred
// would find another token than the definition's. A weight costs 20
// instructions of 64 bits, each as long as one of 32.
#include <math.h>

#include "mh_kvtree.cuh"

namespace mh {
namespace {

constexpr int kThreads = 256;           // of a block that reads logits
constexpr int kMaxSlices = 256;         // of a row
constexpr int kWalk = 1024, kWalkWaves = kWalk / 64;

// What a slice of a row's logits adds up to.
struct __attribute__((aligned(16))) Part {
    double z;       // sum of 2^((x - m) heat) (0: no token, NaN: a row without probabilities); temp <= 0: 0 or NaN
    float m;        // largest logit
    int32_t at;     // its first token (temp <= 0)
};

// A sequence whose last row k_vf_rest has to look at.
struct __attribute__((aligned(16))) Last {
    double alpha, inv;   // max(w inv - alpha q, 0)
    float m;
    int32_t row;         // -1: none
    unsigned done;       // blocks that have left their sums
    int32_t pad;
};

struct VfArgs {
    const float *x, *q, *u;
    const int32_t *row0, *parent, *token;
    int32_t *n_kept, *kept, *next;
    Part *part;       // [n_rows][slices]
    Last *last;       // [n_seqs]
    double *rest;     // [n_seqs][rslices]
    unsigned *err;
    int64_t ld, ldq, V, slice, rslice;
    double heat;      // log2(e) / temp
    int n_seqs, n_rows, max_rows, slices, rslices;
};

enum { GREEDY = 0, CHOSEN = 1, DRAWN = 2 };   // temp <= 0; drafts without probabilities; with

__device__ __forceinline__ double wave_sum64(double v) {
#pragma unroll
    for (int o = 32; o; o >>= 1) v += __shfl_xor(v, o, 64);
    return v;
}

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
        for (int j = 0; j < 4; ++j) v[j] = i + j < stop ? x[i + j] : pad;
    }
}
__device__ __forceinline__ bool aligned16(const void *p) { return (uintptr_t)p % 16 == 0; }

// A block per slice of a row (blockIdx.y): its largest logit and its sum of
// weights, or its first largest token.
template <bool FIRST, int E>
__global__ void __launch_bounds__(kThreads, 4) k_vf_part(VfArgs A, int first) {
    constexpr int CHUNK = kThreads * E;
    __shared__ double sz[kThreads / 64];
    __shared__ float sm[kThreads / 64];
    __shared__ int sa[kThreads / 64];
    const int t = threadIdx.x, wave = t >> 6;
    const int64_t row = first + blockIdx.y, begin = (int64_t)blockIdx.x * A.slice, stop = min(begin + A.slice, A.V);
    if (A.row0 && (row < A.row0[0] || row >= A.row0[A.n_seqs])) return;   // of no sequence
    const float *x = A.x + row * A.ld;
    const bool vec = aligned16(x);
    float m = -INFINITY, nx[E], v[E];
    double z0 = 0.0, z1 = 0.0;
    bool odd = false;
    int at = INT32_MAX;
    auto load = [&](int64_t c0) {
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
    const bool bad = __syncthreads_or(odd);
    if ((t & 63) == 0) sz[wave] = z, sm[wave] = M, sa[wave] = at;
    __syncthreads();
    if (t) return;
    Part p{0.0, sm[0], sa[0]};
    for (int w = 1; w < kThreads / 64; ++w)
        if (sm[w] > p.m || (sm[w] == p.m && sa[w] < p.at)) p.m = sm[w], p.at = sa[w];
    if (!FIRST)
        for (int w = 0; w < kThreads / 64; ++w) p.z += sz[w] * weight(sm[w], p.m, A.heat);
    if (bad) p.z = NAN;
    A.part[row * A.slices + blockIdx.x] = p;
}

// The first of a block's threads at which the running sum of v passes `want`
// (and v > 0; if rounding leaves none, the last with v > 0; -1: none has), and
// the sum before it. `before` and the result are the same for all threads.
template <int THREADS>
__device__ __forceinline__ int find(double v, double want, double *before) {
    constexpr int W = THREADS / 64;
    __shared__ double sum[W], at[THREADS];
    __shared__ int hit[W], some[W];
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
    double run = v;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const double p = __shfl_up(run, o, 64);
        if (lane >= o) run += p;
    }
    __syncthreads();
    if (lane == 63) sum[wave] = run;
    __syncthreads();
    double base = 0.0;
    for (int w = 0; w < wave; ++w) base += sum[w];
    const uint64_t past = __ballot(v > 0.0 && base + run > want), any = __ballot(v > 0.0);
    at[t] = base + run - v;
    if (lane == 0) {
        hit[wave] = past ? wave * 64 + __builtin_ctzll(past) : -1;
        some[wave] = any ? wave * 64 + 63 - __builtin_clzll(any) : -1;
    }
    __syncthreads();
    int r = -1, last = -1;
    for (int w = 0; w < W; ++w) {
        if (r < 0) r = hit[w];
        if (some[w] >= 0) last = some[w];
    }
    r = r < 0 ? last : r;
    *before = r < 0 ? 0.0 : at[r];
    __syncthreads();
    return r;
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

// The first token of [a, b) at which the running sum of rest(token) passes
// `want`: a run of tokens each thread, then the run's own. (Written to `out` by
// one thread.)
template <int THREADS, class F>
__device__ __forceinline__ void pick(int64_t a, int64_t b, double want, F rest4, int32_t *out) {
    const int64_t per = ((b - a + THREADS - 1) / THREADS + 3) / 4 * 4, from = a + threadIdx.x * per, to = min(from + per, b);
    double v = 0.0;
    for (int64_t i = from; i < to; i += 4) {
        double r[4];
        rest4(i, to, r);
        v += (r[0] + r[1]) + (r[2] + r[3]);
    }
    double before;
    const int t = find<THREADS>(v, want, &before);
    if ((int)threadIdx.x != max(t, 0)) return;
    double run = before;
    int32_t last = (int32_t)min(from, b - 1);
    for (int64_t i = from; i < to; i += 4) {
        double r[4];
        rest4(i, to, r);
        for (int j = 0; j < 4; ++j) {
            if (!(r[j] > 0.0)) continue;
            run += r[j];
            last = (int32_t)(i + j);
            if (run > want) {
                *out = last;
                return;
            }
        }
    }
    *out = last;
}

// A block per sequence. A wave a row joins the row's slices; lane i of every
// wave then has row i of the tree, and all walk down it alike: the drafts that
// follow the current row are bits of a ballot. At the end the slices of the
// last row, without what refused drafts took of them, tell the one in which
// the running sum passes the draw.
template <int MODE>
__global__ void __launch_bounds__(kWalk) k_vf_walk(VfArgs A) {
    __shared__ int arg[kTreeRows], gone[kTreeRows];
    __shared__ float top[kTreeRows];
    __shared__ double zs[kTreeRows];
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6, s = blockIdx.x;
    const int r0 = A.row0 ? A.row0[s] : s, r1 = A.row0 ? A.row0[s + 1] : s + 1, n = r1 - r0;
    const bool ok = r0 >= 0 && r1 >= r0 && r1 <= A.n_rows && n <= A.max_rows;
    if (!ok && t == 0) raise_err(A.err);
    int32_t *const kept = A.kept + (int64_t)s * A.max_rows;
    if (MODE == DRAWN && t == 0) A.last[s].row = -1, A.last[s].done = 0;
    if (!ok || n == 0) {
        if (t < A.max_rows) kept[t] = -1;
        if (t == 0) A.n_kept[s] = 0, A.next[s] = -1;
        return;
    }
    int par = -1, tok = -1;
    float u = 0.f, x = -INFINITY, qc = 0.f;
    if (lane < n) {
        par = A.parent ? A.parent[r0 + lane] : lane - 1;
        tok = A.token[r0 + lane];
        u = A.u[r0 + lane];
        if (par < -1 || par >= lane) {
            raise_err(A.err);
            par = -1;
        }
        if (par >= 0 && tok >= 0 && tok < A.V) {
            if (MODE != GREEDY) x = A.x[(int64_t)(r0 + par) * A.ld + tok];
            if (MODE == DRAWN) qc = A.q[(int64_t)(r0 + par) * A.ldq + tok];
        } else {
            par = -1;   // (passed over)
        }
    }
    for (int r = wave; r < n; r += kWalkWaves) {
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
                z += p[k].z * weight(p[k].m, M, A.heat);
            }
        }
        z = wave_sum64(z);
        if (MODE == GREEDY) at = wave_min(at);
        if (lane == 0) top[r] = M, zs[r] = z, arg[r] = z != z || M == -INFINITY ? -1 : at;
    }
    __syncthreads();
    const double w = MODE != GREEDY && par >= 0 ? weight(x, top[par], A.heat) : 0.0;
    int cur = 0, n_kept = 1, at = 0;   // at: the last row that was looked at
    double z = zs[0], inv = 1.0 / z;
    uint64_t out = 0;                  // the refused drafts after the current row
    double off = 0.0;                  // what they took (CHOSEN)
    double alpha = 0.0, left = 1.0;    // max(w / z - alpha q, 0) and its sum (DRAWN)
    bool stale = false;                // `left` is of an earlier alpha
    const float *xr = nullptr, *qr = nullptr;
    bool xv = false, qv = false;
    float m = 0.f;
    auto on_row = [&]() {
        xr = A.x + (int64_t)(r0 + cur) * A.ld;
        xv = aligned16(xr);
        m = top[cur];
        if (MODE == DRAWN) {
            qr = A.q + (int64_t)(r0 + cur) * A.ldq;
            qv = aligned16(qr);
        }
    };
    on_row();
    int n_gone = 0;
    auto rest4 = [&](int64_t i, int64_t to, double *r) {
        float a[4], b[4];
        load4(xr, i, to, xv, -INFINITY, a);
        if (MODE == DRAWN && alpha > 0.0) {
            load4(qr, i, to, qv, 0.f, b);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const double d = __builtin_fma(-alpha, (double)b[j], weight(a[j], m, A.heat) * inv);
                r[j] = d > 0.0 ? d : 0.0;
            }
            return;
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) r[j] = weight(a[j], m, A.heat);
        for (int k = 0; k < n_gone; ++k)
#pragma unroll
            for (int j = 0; j < 4; ++j) r[j] = gone[k] == i + j ? 0.0 : r[j];
    };
    auto sum_of = [&](int64_t a, int64_t b) {
        double v = 0.0;
        for (int64_t i = a + 4 * t; i < b; i += 4 * kWalk) {
            double r[4];
            rest4(i, b, r);
            v += (r[0] + r[1]) + (r[2] + r[3]);
        }
        return block_sum64<kWalk>(v);
    };
    for (;;) {
        const uint64_t after = __ballot(par == cur) & ~((2ull << at) - 1);   // (2 << 63: 0, none after)
        if (!after) break;
        const int i = __builtin_amdgcn_readfirstlane(__builtin_ctzll(after)), c = __shfl(tok, i, 64);
        bool yes;
        if (MODE == GREEDY) {
            yes = c == arg[cur];
        } else if (MODE == CHOSEN) {
            const bool again = __ballot((out >> lane & 1) && tok == c) != 0;
            const double wc = __shfl(w, i, 64);
            yes = !again && (double)__shfl(u, i, 64) * (z - off) < wc;
            if (!again) off += wc;
        } else {
            if (stale) {
                left = sum_of(0, A.V);
                stale = false;
            }
            const double qd = __shfl(qc, i, 64), d = __builtin_fma(-alpha, qd, __shfl(w, i, 64) * inv);
            yes = (double)__shfl(u, i, 64) * qd * left < (d > 0.0 ? d : 0.0);
            alpha += left;
            stale = true;
        }
        at = i;
        if (!yes) {
            out |= 1ull << i;
            continue;
        }
        if (t == 0) kept[n_kept] = i;
        ++n_kept;
        cur = i;
        z = zs[cur];
        inv = 1.0 / z;
        out = 0;
        off = alpha = 0.0;
        left = 1.0;
        stale = false;
        on_row();
    }
    if (t == 0) kept[0] = 0, A.n_kept[s] = n_kept;
    if (t >= n_kept && t < A.max_rows) kept[t] = -1;
    if (MODE == GREEDY || !(z > 0.0)) {   // (NaN too)
        if (t == 0) A.next[s] = MODE == GREEDY ? arg[cur] : -1;
        return;
    }
    const float u0 = __shfl(u, 0, 64);
    if (MODE == DRAWN && alpha > 0.0) {
        if (t == 0) {
            Last &l = A.last[s];
            l.alpha = alpha;
            l.inv = inv;
            l.m = m;
            l.row = r0 + cur;
        }
        return;
    }
    // the row's slices without the refused tokens
    if (MODE == CHOSEN && out) {
        n_gone = __popcll(out);
        if (wave == 0 && (out >> lane & 1)) gone[__popcll(out & ((1ull << lane) - 1))] = tok;
    }
    __shared__ double share[kMaxSlices];
    __shared__ int again[kMaxSlices];
    __syncthreads();
    double v = 0.0;
    for (int pass = 0; pass < 2; ++pass) {   // (the second: rounding left nothing, the row's own probabilities)
        if (t < kMaxSlices) {
            double all = 0.0;
            if (t < A.slices) {
                const Part p = A.part[(int64_t)(r0 + cur) * A.slices + t];
                all = p.z * weight(p.m, m, A.heat);
            }
            double less = all;
            for (int k = 0; k < n_gone; ++k) {
                bool twice = false;
                for (int j = 0; j < k; ++j) twice |= gone[j] == gone[k];
                if (!twice && gone[k] / A.slice == t) less -= weight(xr[gone[k]], m, A.heat);
            }
            share[t] = less;
            again[t] = less < all * 0x1p-10;   // (too little of it to be a difference: added up again)
        }
        __syncthreads();
        for (int k = 0; k < n_gone; ++k) {
            const int sl = (int)(gone[k] / A.slice);
            if (!again[sl]) continue;
            const double f = sum_of(sl * A.slice, min((sl + 1) * A.slice, A.V));
            if (t == 0) share[sl] = f, again[sl] = 0;
            __syncthreads();
        }
        v = t < kMaxSlices ? share[t] : 0.0;
        const double sum = block_sum64<kWalk>(v);
        if (sum > 0.0) {
            double before;
            const double want = (double)u0 * sum;
            const int sl = find<kWalk>(v, want, &before);
            pick<kWalk>(sl * A.slice, min((sl + 1) * A.slice, A.V), want - before, rest4, A.next + s);
            return;
        }
        n_gone = 0;
        __syncthreads();
    }
    if (t == 0) A.next[s] = -1;
}

// A block per slice of the last row of a sequence that ends with refusals:
// the slice's sum of max(p - alpha q, 0). The block that finishes last finds
// the token (the counter only tells which that is; sums are added in the
// slices' order).
__global__ void __launch_bounds__(kThreads) k_vf_rest(VfArgs A, int first) {
    const int s = first + blockIdx.y, t = threadIdx.x;
    Last *const l = A.last + s;
    const int row = l->row;
    if (row < 0) return;
    const double inv = l->inv;
    double alpha = l->alpha;
    const float m = l->m, *xr = A.x + (int64_t)row * A.ld, *qr = A.q + (int64_t)row * A.ldq;
    const bool xv = aligned16(xr), qv = aligned16(qr);
    auto rest4 = [&](int64_t i, int64_t to, double *r) {
        float a[4], b[4];
        load4(xr, i, to, xv, -INFINITY, a);
        load4(qr, i, to, qv, 0.f, b);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const double w = weight(a[j], m, A.heat) * inv, d = alpha > 0.0 ? __builtin_fma(-alpha, (double)b[j], w) : w;   // (q may be a NaN)
            r[j] = d > 0.0 ? d : 0.0;
        }
    };
    auto sum_of = [&](int64_t a, int64_t b) {
        double v = 0.0;
        for (int64_t i = a + 4 * t; i < b; i += 4 * kThreads) {
            double r[4];
            rest4(i, b, r);
            v += (r[0] + r[1]) + (r[2] + r[3]);
        }
        return block_sum64<kThreads>(v);
    };
    double *const rest = A.rest + (int64_t)s * A.rslices;
    const int64_t begin = (int64_t)blockIdx.x * A.rslice;
    const double mine = sum_of(begin, min(begin + A.rslice, A.V));
    __shared__ bool final;
    if (t == 0) {
        __hip_atomic_store(rest + blockIdx.x, mine, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        final = __hip_atomic_fetch_add(&l->done, 1u, __ATOMIC_ACQ_REL, __HIP_MEMORY_SCOPE_AGENT) == (unsigned)A.rslices - 1;
    }
    __syncthreads();
    if (!final) return;
    const double want0 = (double)A.u[A.row0 ? A.row0[s] : s];
    double v = t < A.rslices ? __hip_atomic_load(rest + t, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) : 0.0;
    double sum = block_sum64<kThreads>(v), before;
    if (!(sum > 0.0)) {   // rounding left nothing: the row's own probabilities
        alpha = 0.0;
        for (int k = 0; k < A.rslices; ++k) {
            const double f = sum_of(k * A.rslice, min((k + 1) * A.rslice, A.V));
            if (t == k) v = f;
        }
        sum = block_sum64<kThreads>(v);
    }
    const int sl = max(find<kThreads>(v, want0 * sum, &before), 0);
    pick<kThreads>(sl * A.rslice, min((sl + 1) * A.rslice, A.V), want0 * sum - before, rest4, A.next + s);
}

// How n rows are cut: chunks of 4 tokens a thread where chunks of 16 would be
// fewer than the 256 CUs, then into the slices (at most 256 of a row) whose
// blocks end soonest: rounds of kResident blocks, each as long as its chunks
// and what a block costs beside them.
constexpr int kResident = 4 * 256, kExtra = 3;
struct Cut {
    int E, slices;
    int64_t slice;
};
Cut cut(int n, int64_t V) {
    Cut c;
    c.E = (int64_t)n * V < (int64_t)256 * kThreads * 16 ? 4 : 16;
    const int64_t chunk = kThreads * c.E, chunks = (V + chunk - 1) / chunk;
    int64_t best = INT64_MAX, per = chunks;
    for (int64_t s = 1; s <= std::min<int64_t>(kMaxSlices, chunks); ++s) {
        const int64_t k = (chunks + s - 1) / s, blocks = (int64_t)std::max(n, 1) * ((chunks + k - 1) / k);
        const int64_t cost = (blocks + kResident - 1) / kResident * (k + kExtra);
        if (cost < best) best = cost, per = k;
    }
    c.slice = per * chunk;
    c.slices = (int)((V + c.slice - 1) / c.slice);
    return c;
}

uint64_t part_bytes(uint64_t n_rows, int64_t V) { return std::max<uint64_t>(n_rows, 1) * std::min<int64_t>(kMaxSlices, (V + 1023) / 1024) * sizeof(Part); }
uint64_t ws_bytes_for(uint64_t n_seqs, uint64_t n_rows, int64_t V) {
    return part_bytes(n_rows, V) + n_seqs * (sizeof(Last) + 8 * (uint64_t)kMaxSlices);
}

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
    const uint64_t xb = n ? 4 * ((n - 1) * d->ld + d->vocab) : 0, qb = n && d->q ? 4 * ((n - 1) * d->ldq + d->vocab) : 0;
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
    const Cut c = cut(d->n_rows, d->vocab), r = cut(d->n_seqs, d->vocab);
    uint8_t *const after = (uint8_t *)ws + part_bytes(n, d->vocab);
    const VfArgs A{d->logits, q ? d->q : nullptr, d->u, d->row0, d->parent, d->token, n_kept, kept, next, (Part *)ws, (Last *)after,
                   (double *)(after + ns * sizeof(Last)), flag, d->ld, d->ldq, d->vocab, c.slice, r.slice,
                   greedy ? 0.0 : 1.4426950408889634 / (double)d->temp, d->n_seqs, d->n_rows, d->max_rows, c.slices, r.slices};
    for (int row = 0; row < d->n_rows; row += 32768) {   // (a grid's second axis ends at 65535)
        const dim3 grid((unsigned)c.slices, (unsigned)std::min(32768, d->n_rows - row));
        const bool few = c.E == 4;
        if (greedy) few ? launch_part<true, 4>(A, grid, row) : launch_part<true, 16>(A, grid, row);
        else few ? launch_part<false, 4>(A, grid, row) : launch_part<false, 16>(A, grid, row);
    }
    const dim3 seqs((unsigned)d->n_seqs);
    if (greedy) MH_LAUNCH("verify_walk", k_vf_walk<GREEDY>, seqs, dim3(kWalk), 0, stream(), A);
    else if (!q) MH_LAUNCH("verify_walk", k_vf_walk<CHOSEN>, seqs, dim3(kWalk), 0, stream(), A);
    else MH_LAUNCH("verify_walk", k_vf_walk<DRAWN>, seqs, dim3(kWalk), 0, stream(), A);
    for (int s = 0; q && s < d->n_seqs; s += 32768)
        MH_LAUNCH("verify_rest", k_vf_rest, dim3((unsigned)r.slices, (unsigned)std::min(32768, d->n_seqs - s)), dim3(kThreads), 0, stream(), A, s);
    return hip_check(hipGetLastError(), "verify launch");
}

}  // extern "C"
