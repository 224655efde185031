// mh_logprobs.hip — log probabilities of given tokens, the entropy and the
// most probable tokens of rows of logits (mh_logprobs_dev).
#include <math.h>

#include "mh_internal.h"

namespace mh {
namespace {

constexpr int kLpTop = 64, kThreads = 256;
constexpr int kCap = 512;        // candidates of a chunk that are ranked at once
constexpr int kMaxSlices = kThreads;  // of a row: a thread a slice where they are joined

struct LpArgs {
    const float *x;
    const int32_t *ids;
    float *lp, *entropy, *top_lp;
    int32_t *top_id;
    float *part;        // [n][slices][4]: maximum, sum, weighted sum, 1 if a NaN
    uint64_t *keys;     // [n][slices][top]: the slices' alternatives, best first (0: none)
    int64_t ld, V, slice;   // slice: tokens a block takes of a row, a multiple of its chunk
    int m, top, slices;
};

constexpr float kLog2e = 1.44269504088896341f;

// x - m for x <= m, at least -200, where e^(x - m) is 0 in 32 bits: its
// products with sums stay finite, -inf (or the type's lowest value) included,
// and both -inf (no token so far: sums of 0) give -200 too.
__device__ __forceinline__ float shift(float x, float m) { return fmaxf(x - m, -200.f); }

// Order of the alternatives: larger logits first (-0 as 0, NaN behind
// everything), then lower ids; never 0.
__device__ __forceinline__ uint32_t order32(float x) {
    uint32_t u = __float_as_uint(x == 0.f ? 0.f : x);
    u = u >> 31 ? ~u : u | 0x80000000u;
    return x != x ? 0u : u;
}
__device__ __forceinline__ uint64_t order64(float x, uint32_t id) { return (uint64_t)order32(x) << 32 | (uint32_t)~id; }
__device__ __forceinline__ float order_value(uint32_t u) {
    return u ? __uint_as_float(u >> 31 ? u & 0x7fffffffu : ~u) : __uint_as_float(0x7fc00000u);
}

__device__ __forceinline__ float block_max(float v, float *red) {
    v = wave_max(v);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    return fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
}
__device__ __forceinline__ float block_sum(float v, float *red) {
    v = wave_sum_dpp(v);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    return (red[0] + red[1]) + (red[2] + red[3]);
}

// The largest u for which at least `want` of the wave's lanes have k >= u
// (bit by bit from the top; 0 if fewer than `want` lanes have any).
__device__ __forceinline__ uint32_t wave_kth(uint32_t k, int want) {
    uint32_t u = 0;
    for (int bit = 31; bit >= 0; --bit) {
        const uint32_t c = u | 1u << bit;
        if (__popcll(__ballot(k >= c)) >= want) u = c;
    }
    return u;
}

// The best `top` of the n keys in `cand` and the `have` in `best`, in order,
// into `next` (0 behind the last): each key's rank is the number of greater
// ones. All keys differ.
__device__ __forceinline__ void rank_keys(const uint64_t *cand, int n, const uint64_t *best, int have, int top, uint64_t *next) {
    for (int i = threadIdx.x; i < n + have; i += kThreads) {
        const uint64_t k = i < n ? cand[i] : best[i - n];
        int r = 0;
#pragma unroll 8
        for (int j = 0; j < n; ++j) r += cand[j] > k;   // (eight reads on their way at once)
#pragma unroll 8
        for (int j = 0; j < have; ++j) r += best[j] > k;
        if (r < top) next[r] = k;
    }
    if (n + have + (int)threadIdx.x < top) next[n + have + threadIdx.x] = 0;
}

// A block per slice of a row: chunks of 256 * E tokens in registers, each
// thread's running maximum, sum and weighted sum, and the slice's best
// tokens. A chunk's candidates are the tokens above the running list's last
// one; the first chunk (and one with too many) takes as bound the `top`-th
// largest of a wave's 64 thread maxima, which `top` tokens reach. Where even
// that leaves too many (equal logits, NaNs), they are picked one by one.
// 400 rows of 201088 logits (322 MB) with 5 alternatives 68 us = 4.7 TB/s, with
// 20 of them 85 us: one chunk is on its way beside the one in registers, and
// the alternatives' exchanges stand between loads (a long read of weights by
// this library's GEMVs runs at 6.1 TB/s, which would be 53 us). One row (0.8 MB)
// 7 us, by the chunk's exchanges.
template <int E>
__global__ void __launch_bounds__(kThreads, 4) k_lp_part(LpArgs A) {
    constexpr int CHUNK = kThreads * E;
    __shared__ float red[4];
    __shared__ uint64_t cand[kCap], lists[2][kLpTop], kred[4];
    __shared__ uint32_t bound[4];
    __shared__ int cnt[3];
    const int t = threadIdx.x;
    const int64_t row = blockIdx.y, begin = (int64_t)blockIdx.x * A.slice, stop = min(begin + A.slice, A.V);
    const float *x = A.x + row * A.ld;
    const bool vec = (uintptr_t)x % 16 == 0;
    if (t < 3) cnt[t] = 0;
    float m = -INFINITY, z = 0.f, w = 0.f;
    bool nan = false;
    int have = 0, cur = 0;
    float last = 0.f;   // the list's last logit once it is full
    float v[E], nx[E];
    auto load = [&](int64_t c0) {
        if (vec && c0 + CHUNK <= stop) {   // (all in one block: none waits for another)
#pragma unroll
            for (int j = 0; j < E / 4; ++j) {
                const float4 f = *(const float4 *)(x + c0 + 4 * (j * kThreads + t));
                nx[4 * j] = f.x;
                nx[4 * j + 1] = f.y;
                nx[4 * j + 2] = f.z;
                nx[4 * j + 3] = f.w;
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
    __syncthreads();
    int it = 0;
    for (int64_t c0 = begin; c0 < stop; c0 += CHUNK, it = it == 2 ? 0 : it + 1) {
#pragma unroll
        for (int j = 0; j < E; ++j) v[j] = nx[j];
        if (c0 + CHUNK < stop) load(c0 + CHUNK);
        float tm = -INFINITY;
        bool odd = false;
#pragma unroll
        for (int j = 0; j < E; ++j) {
            tm = fmaxf(tm, v[j]);
            odd |= v[j] != v[j];
        }
        nan |= odd;
        if (tm > m) {   // e^(m - tm) of the old sums; (w + (m - tm) z) for the weighted one
            const float dm = shift(m, tm), f = __builtin_amdgcn_exp2f(dm * kLog2e);
            w = f * __builtin_fmaf(dm, z, w);
            z *= f;
            m = tm;
        }
        const float ms = m == -INFINITY ? 0.f : m;
#pragma unroll
        for (int j = 0; j < E; ++j) {
            const float d = shift(v[j], ms), e = __builtin_amdgcn_exp2f(d * kLog2e);
            z += e;
            w = __builtin_fmaf(e, d, w);
        }
        if (!A.top) continue;
        // tokens of this thread: value v[j], id c0 + 4 * (j / 4 * 256 + t) + j % 4
        auto id = [&](int j) { return (uint32_t)(c0 + 4 * (j / 4 * kThreads + t) + j % 4); };
        auto push = [&](float lo, bool equal) {
            if (!(tm > lo || (equal && tm == lo))) return;
#pragma unroll
            for (int j = 0; j < E; ++j)
                if ((v[j] > lo || (equal && v[j] == lo)) && id(j) < stop) {
                    const int at = atomicAdd(&cnt[it], 1);
                    if (at < kCap) cand[at] = order64(v[j], id(j));
                }
        };
        bool search = have < A.top;
        if (!search) push(last, false);
        // (a list that ends with a NaN: any token of the chunk passes it)
        bool slow = __syncthreads_or(odd) || (!search && last != last);
        int n = cnt[it];
        if (t == 0) cnt[it == 0 ? 2 : it - 1] = 0;   // the last chunk's, the next but one's
        if (!slow && !search && n == 0) continue;
        if (!slow && !search && n > kCap) {
            __syncthreads();
            if (t == 0) cnt[it] = 0;
            search = true;
        }
        if (!slow && search) {
            const uint32_t u = wave_kth(tm == -INFINITY ? 0u : order32(tm), A.top);
            if ((t & 63) == 0) bound[t >> 6] = u;
            __syncthreads();
            const uint32_t b = max(max(bound[0], bound[1]), max(bound[2], bound[3]));
            push(b ? order_value(b) : -INFINITY, true);
            __syncthreads();
            n = cnt[it];
            slow = n > kCap;
        }
        if (slow) {
            // one by one, the list's own among them
            uint64_t top_key = ~0ull;
            int k = 0;
            for (; k < A.top; ++k) {
                uint64_t best = 0;
#pragma unroll
                for (int j = 0; j < E; ++j) {
                    const uint64_t key = id(j) < stop ? order64(v[j], id(j)) : 0;
                    if (key < top_key && key > best) best = key;
                }
                if (t < have && lists[cur][t] < top_key && lists[cur][t] > best) best = lists[cur][t];
                for (int o = 32; o; o >>= 1) {
                    const uint64_t key = __shfl_xor((unsigned long long)best, o, 64);
                    best = key > best ? key : best;
                }
                __syncthreads();
                if ((t & 63) == 0) kred[t >> 6] = best;
                __syncthreads();
                for (int o = 0; o < 4; ++o) best = kred[o] > best ? kred[o] : best;
                if (t == 0) lists[1 - cur][k] = best;
                top_key = best;
                if (best == 0) {   // fewer than top tokens so far
                    for (int i = k + t; i < A.top; i += kThreads) lists[1 - cur][i] = 0;
                    break;
                }
            }
            have = k;
        } else {
            rank_keys(cand, n, lists[cur], have, A.top, lists[1 - cur]);
            have = min(A.top, n + have);   // (short only where the tokens so far are fewer than top)
        }
        __syncthreads();
        cur = 1 - cur;
        if (have == A.top) last = order_value((uint32_t)(lists[cur][A.top - 1] >> 32));
    }
    const float M = block_max(m, red), dm = shift(m, M), f = __builtin_amdgcn_exp2f(dm * kLog2e);
    w = f * __builtin_fmaf(dm, z, w);
    z = block_sum(f * z, red);
    w = block_sum(w, red);
    const int any = __syncthreads_or(nan);
    const int64_t at = row * A.slices + blockIdx.x;
    if (t == 0) *(float4 *)&A.part[4 * at] = make_float4(M, z, w, any ? 1.f : 0.f);
    if (t < A.top) A.keys[at * A.top + t] = lists[cur][t];
}

// A block per row: the slices' sums and lists joined, the given tokens. A
// thread holds a slice's sums and the first kHeld of its list, so that one
// trip to memory brings nearly all that is needed: 5.5 us for one row of 197
// slices, 6.3 for 400 rows. (All keys in one flat read: the same.) A lane walks
// what its slice's list has past those one by one: in rows of one slice, where
// the list is the answer, 32 alternatives take 9 us and 4 take 6 (4 rows of 4000).
constexpr int kHeld = 4;
__global__ void __launch_bounds__(kThreads) k_lp_join(LpArgs A) {
    __shared__ float red[4];
    __shared__ uint64_t cand[kCap], list[kLpTop];
    __shared__ uint64_t kred[4];
    __shared__ uint32_t heads[kMaxSlices], bound;
    __shared__ int cnt;
    const int t = threadIdx.x;
    const int64_t row = blockIdx.x;
    const float *x = A.x + row * A.ld;
    const uint64_t *keys = A.keys + row * A.slices * A.top, *mine = keys + (int64_t)t * A.top;
    float4 p = make_float4(-INFINITY, 0.f, 0.f, 0.f);
    uint64_t held[kHeld];
#pragma unroll
    for (int j = 0; j < kHeld; ++j) held[j] = t < A.slices && j < A.top ? mine[j] : 0;
    if (t < A.slices) p = *(const float4 *)&A.part[4 * (row * A.slices + t)];
    int id = -1;
    float want = 0.f;
    if (t < A.m) {
        id = A.ids[row * A.m + t];
        if (id >= 0 && id < A.V) want = x[id];
    }
    if (t == 0) cnt = 0;
    const float M = block_max(p.x, red), dm = shift(p.x, M), f = __builtin_amdgcn_exp2f(dm * kLog2e);
    const bool none = M == -INFINITY, bad = __syncthreads_or(p.w != 0.f) || M == INFINITY;
    const float w = block_sum(f * __builtin_fmaf(dm, p.y, p.z), red), z = block_sum(f * p.y, red);
    const float lz = logf(z);
    auto lp = [&](float v) { return bad ? NAN : none ? -INFINITY : (v - M) - lz; };
    for (int j = t; j < A.m; j += kThreads) {
        if (j != t) {
            id = A.ids[row * A.m + j];
            if (id >= 0 && id < A.V) want = x[id];
        }
        A.lp[row * A.m + j] = id >= 0 && id < A.V ? lp(want) : bad ? NAN : -INFINITY;
    }
    if (t == 0 && A.entropy) A.entropy[row] = bad ? NAN : none ? 0.f : lz - w / z;
    if (!A.top) return;
    // a bound that `top` keys reach: of the lists' entries number d (top <= slices * (d + 1)), the k-th largest
    // with k (d + 1) >= top
    const int d = (A.top - 1) / A.slices, k = (A.top + d) / (d + 1);
    heads[t] = t < A.slices ? (uint32_t)((d < kHeld ? held[0] : mine[d]) >> 32) : 0u;
#pragma unroll
    for (int j = 1; j < kHeld; ++j)
        if (j == d) heads[t] = (uint32_t)(held[j] >> 32);
    __syncthreads();
    if (t < 64) {
        uint32_t h[kMaxSlices / 64];
#pragma unroll
        for (int j = 0; j < kMaxSlices / 64; ++j) h[j] = heads[t + 64 * j];
        uint32_t u = 0;
        for (int bit = 31; bit >= 0; --bit) {
            const uint32_t c = u | 1u << bit;
            int n = 0;
#pragma unroll
            for (int j = 0; j < kMaxSlices / 64; ++j) n += __popcll(__ballot(h[j] >= c));
            if (n >= k) u = c;
        }
        if (t == 0) bound = u;
    }
    __syncthreads();
    const uint32_t lo = bound;
    auto push = [&](uint64_t key) {
        const int at = atomicAdd(&cnt, 1);
        if (at < kCap) cand[at] = key;
    };
    auto in = [&](uint64_t key) { return key && (uint32_t)(key >> 32) >= lo; };
#pragma unroll
    for (int j = 0; j < kHeld; ++j)
        if (in(held[j])) push(held[j]);
    if (t < A.slices && in(held[kHeld - 1]))
        for (int j = kHeld; j < A.top && in(mine[j]); ++j) push(mine[j]);
    __syncthreads();
    const int found = cnt;
    if (found <= kCap) {
        rank_keys(cand, found, cand, 0, A.top, list);
        __syncthreads();
    } else {   // equal logits: one by one
        uint64_t last = ~0ull;
        for (int j = 0; j < A.top; ++j) {
            uint64_t best = 0;
            for (int i = t; i < A.slices * A.top; i += kThreads)
                if (keys[i] < last && keys[i] > best) best = keys[i];
            for (int o = 32; o; o >>= 1) {
                const uint64_t key = __shfl_xor((unsigned long long)best, o, 64);
                best = key > best ? key : best;
            }
            __syncthreads();
            if ((t & 63) == 0) kred[t >> 6] = best;
            __syncthreads();
            for (int o = 0; o < 4; ++o) best = kred[o] > best ? kred[o] : best;
            if (t == 0) list[j] = best;
            last = best;
        }
        __syncthreads();
    }
    if (t < A.top) {
        A.top_id[row * A.top + t] = (int32_t)~(uint32_t)list[t];
        A.top_lp[row * A.top + t] = lp(order_value((uint32_t)(list[t] >> 32)));   // (the logit itself, -0 as 0)
    }
}

// How a call is cut: chunks of 4 tokens a thread where chunks of 16 would be
// fewer than the 256 CUs (20 alternatives, us with 4 / 16: 1 row of 201088
// 12.7 / 14.6, 4 13.8 / 14.8, 8 16.5 / 15.0, 400 143 / 90; 16 of 32000 13.3 /
// 16.8, 64 17.9 / 18.6), then into the slices (at most 256 of a row) whose
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

uint64_t ws_bytes_for(uint64_t lists, int top) { return lists * (16 + 8 * (uint64_t)top) + 16; }

// Slices' sums and lists that any call of at most n rows of at most V tokens
// leaves: chunks of 4 are taken where n * V < 2^20, so that n rows of
// ceil(V / 1024) of them are fewer than n + 1024; of chunks of 16 a row has
// ceil(V / 4096). (The cuts themselves are not monotone: 5 rows of 201088 make
// 985 slices, 6 make 300.)
uint64_t most_lists(int n, int64_t V) {
    auto slices = [V](int E) { return std::min<int64_t>(kMaxSlices, (V + kThreads * E - 1) / (kThreads * E)); };
    return (uint64_t)std::max(std::min(n * slices(4), (int64_t)n + 1024), n * slices(16));
}

int validate(int n, int64_t V, int top, const char *what) {
    if (n < 0 || n >= (1 << 24)) return fail(MH_E_ARG, "%s: %d rows", what, n);
    if (V < 1 || V > (1 << 30)) return fail(MH_E_ARG, "%s: vocabulary of %lld tokens", what, (long long)V);
    if (top < 0 || top > kLpTop || top > V) return fail(MH_E_ARG, "%s: %d alternatives (at most %d, and the vocabulary)", what, top, kLpTop);
    return MH_OK;
}

}  // namespace
}  // namespace mh

using namespace mh;

extern "C" {

int mh_logprobs_ws(int n, int64_t V, int top, uint64_t *bytes) {
    clear_error();
    MH_TRY(validate(n, V, top, "mh_logprobs_ws"));
    if (!bytes) return fail(MH_E_ARG, "mh_logprobs_ws: NULL result");
    *bytes = ws_bytes_for(most_lists(n, V), top);
    return MH_OK;
}

int mh_logprobs_dev(const float *logits, int64_t ld, int n, int64_t V, const int32_t *ids, int m, int top, float *lp,
                    float *entropy, int32_t *top_id, float *top_lp, void *ws, uint64_t ws_bytes) {
    const char *what = "mh_logprobs_dev";
    clear_error();
    MH_TRY(validate(n, V, top, what));
    const Cut c = cut(n, V);
    const uint64_t need = ws_bytes_for((uint64_t)n * c.slices, top);   // (of this call: mh_logprobs_ws covers the smaller ones too)
    if (!logits || !ws) return fail(MH_E_ARG, "%s: NULL logits or workspace", what);
    if (ld < V || ld > ((int64_t)1 << 40)) return fail(MH_E_ARG, "%s: rows of %lld floats, %lld tokens", what, (long long)ld, (long long)V);
    uint64_t xb;
    MH_TRY(rows_bytes(n, ld, V, &xb, what));
    if (m < 0 || m > (1 << 20) || (m && (!ids || !lp))) return fail(MH_E_ARG, "%s: %d tokens a row without ids or lp", what, m);
    if (top && (!top_id || !top_lp)) return fail(MH_E_ARG, "%s: alternatives without top_id or top_lp", what);
    if (!m && !top && !entropy) return fail(MH_E_ARG, "%s: nothing wanted", what);
    if (ws_bytes < need) return fail(MH_E_ARG, "%s: a workspace of %llu bytes, %llu needed", what, (unsigned long long)ws_bytes,
                                     (unsigned long long)need);
    if (((uintptr_t)logits | (uintptr_t)ids | (uintptr_t)lp | (uintptr_t)entropy | (uintptr_t)top_id | (uintptr_t)top_lp) % 4 ||
        (uintptr_t)ws % 16)
        return fail(MH_E_ARG, "%s: misaligned argument", what);
    MH_TRY(require_init());
    if (!n) return MH_OK;
    OnDevice here;
    MH_TRY(resolve_here(logits, xb, what));
    if (m) {
        MH_TRY(resolve_here(ids, 4 * (uint64_t)n * m, what));
        MH_TRY(resolve_here(lp, 4 * (uint64_t)n * m, what));
    }
    if (entropy) MH_TRY(resolve_here(entropy, 4 * (uint64_t)n, what));
    if (top) {
        MH_TRY(resolve_here(top_id, 4 * (uint64_t)n * top, what));
        MH_TRY(resolve_here(top_lp, 4 * (uint64_t)n * top, what));
    }
    MH_TRY(resolve_here(ws, need, what));
    const struct {
        const void *p;
        uint64_t n;
    } mem[] = {{ws, need}, {m ? lp : nullptr, 4 * (uint64_t)n * m}, {entropy, 4 * (uint64_t)n}, {top ? top_id : nullptr, 4 * (uint64_t)n * top},
               {top ? top_lp : nullptr, 4 * (uint64_t)n * top}, {m ? ids : nullptr, 4 * (uint64_t)n * m}, {logits, xb}};
    for (int i = 0; i < 5; ++i)   // (what is written, against all)
        for (int j = i + 1; j < 7; ++j)
            if (mem[i].p && mem[j].p && (uintptr_t)mem[i].p < (uintptr_t)mem[j].p + mem[j].n && (uintptr_t)mem[j].p < (uintptr_t)mem[i].p + mem[i].n)
                return fail(MH_E_ARG, "%s: %p overlaps %p", what, mem[i].p, mem[j].p);
    LpArgs A{logits, ids, lp, entropy, top_lp, top_id, (float *)ws, (uint64_t *)((uint8_t *)ws + 16 * (uint64_t)n * c.slices), ld, V, c.slice,
             m, top, c.slices};
    for (int r = 0; r < n; r += 32768) {   // (a grid's second axis ends at 65535)
        LpArgs P = A;
        const int k = std::min(32768, n - r);
        P.x += (int64_t)r * ld;
        P.part += (int64_t)4 * r * c.slices;
        P.keys += (int64_t)r * c.slices * top;
        if (c.E == 4) MH_LAUNCH("logprobs", k_lp_part<4>, dim3((unsigned)c.slices, (unsigned)k), dim3(kThreads), 0, stream(), P);
        else MH_LAUNCH("logprobs", k_lp_part<16>, dim3((unsigned)c.slices, (unsigned)k), dim3(kThreads), 0, stream(), P);
    }
    MH_LAUNCH("logprobs_join", k_lp_join, dim3((unsigned)n), dim3(kThreads), 0, stream(), A);
    return hip_check(hipGetLastError(), "logprobs launch");
}

}  // extern "C"
