// mh_verify.hip — which drafted tokens the target's probabilities keep, and the
// token after them (mh_verify_dev).
#include <math.h>

#include "mh_kvtree.cuh"

namespace mh {
namespace {

constexpr int kThreads = 256;           // of a block that reads logits
constexpr int kMaxSlices = 256;         // of a row
constexpr int kWalk = 1024, kWalkWaves = kWalk / 64;

// What a slice of a row's logits adds up to.
struct __attribute__((aligned(16))) Part {
    double z;       // sum of e^((x - m) / temp) (0: no token, NaN: a row without probabilities); temp <= 0: 0 or NaN
    float m;        // largest logit
    int32_t at;     // its first token (temp <= 0)
};

struct VfArgs {
    const float *x, *q, *u;
    const int32_t *row0, *parent, *token;
    int32_t *n_kept, *kept, *next;
    Part *part;     // [n_rows][slices]
    unsigned *err;
    int64_t ld, ldq, V, slice;
    double heat;    // 1 / temp, 0 where temp <= 0
    int n_seqs, n_rows, max_rows, slices;
};

__device__ __forceinline__ double wave_sum64(double v) {
#pragma unroll
    for (int o = 32; o; o >>= 1) v += __shfl_xor(v, o, 64);
    return v;
}

// Weight of logit x beside the largest m of its row: e^((x - m) / temp).
__device__ __forceinline__ double weight(float x, float m, double heat) { return exp(((double)x - (double)m) * heat); }

// A block per slice of a row (blockIdx.y): its largest logit and its sum of
// weights, or its first largest token.
template <bool GREEDY>
__global__ void __launch_bounds__(kThreads) k_vf_part(VfArgs A, int first) {
    __shared__ double sz[kThreads / 64];
    __shared__ float sm[kThreads / 64];
    __shared__ int sa[kThreads / 64];
    const int t = threadIdx.x, wave = t >> 6;
    const int64_t row = first + blockIdx.y, begin = (int64_t)blockIdx.x * A.slice, stop = min(begin + A.slice, A.V);
    if (A.row0 && (row < A.row0[0] || row >= A.row0[A.n_seqs])) return;   // of no sequence
    const float *x = A.x + row * A.ld;
    float m = -INFINITY;
    double z = 0.0;
    bool odd = false;
    int at = INT32_MAX;
    for (int64_t i = begin + t; i < stop; i += kThreads) {
        const float v = x[i];
        odd |= v != v;
        if (v > m) {
            if (!GREEDY) z *= m == -INFINITY ? 0.0 : weight(m, v, A.heat);
            m = v;
            at = (int)i;
        }
        if (!GREEDY && v != -INFINITY) z += weight(v, m, A.heat);
    }
    const float M = wave_max(m);
    if (GREEDY) at = wave_min(m == M && M != -INFINITY ? at : INT32_MAX);
    else z = wave_sum64(m == -INFINITY ? 0.0 : z * weight(m, M, A.heat));
    const bool bad = __syncthreads_or(odd);
    if ((t & 63) == 0) sz[wave] = z, sm[wave] = M, sa[wave] = at;
    __syncthreads();
    if (t) return;
    Part p{0.0, sm[0], sa[0]};
    for (int w = 1; w < kThreads / 64; ++w)
        if (sm[w] > p.m || (sm[w] == p.m && sa[w] < p.at)) p.m = sm[w], p.at = sa[w];
    if (!GREEDY)
        for (int w = 0; w < kThreads / 64; ++w) p.z += sm[w] == -INFINITY ? 0.0 : sz[w] * weight(sm[w], p.m, A.heat);
    if (bad) p.z = NAN;
    A.part[row * A.slices + blockIdx.x] = p;
}

// A block per sequence: the rows' sums joined (a wave a row), the walk down
// the tree (by every thread alike), and the token after it.
template <bool GREEDY>
__global__ void __launch_bounds__(kWalk) k_vf_walk(VfArgs A) {
    __shared__ int par[kTreeRows], tok[kTreeRows], arg[kTreeRows], gone[kTreeRows];
    __shared__ float u[kTreeRows], top[kTreeRows], qc[kTreeRows];
    __shared__ double z[kTreeRows], e[kTreeRows], piece[kWalkWaves];
    __shared__ int pick;
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6, s = blockIdx.x;
    const int r0 = A.row0 ? A.row0[s] : s, r1 = A.row0 ? A.row0[s + 1] : s + 1, n = r1 - r0;
    const bool ok = r0 >= 0 && r1 >= r0 && r1 <= A.n_rows && n <= A.max_rows;
    if (!ok && t == 0) raise_err(A.err);
    int32_t *const kept = A.kept + (int64_t)s * A.max_rows;
    if (!ok || n == 0) {
        if (t < A.max_rows) kept[t] = -1;
        if (t == 0) A.n_kept[s] = 0, A.next[s] = -1;
        return;
    }
    if (t < n) {
        int p = A.parent ? A.parent[r0 + t] : t - 1;
        if (p < -1 || p >= t) {
            raise_err(A.err);
            p = -1;
        }
        par[t] = p;
        tok[t] = A.token[r0 + t];
        u[t] = A.u[r0 + t];
    }
    for (int r = wave; r < n; r += kWalkWaves) {
        const Part *part = A.part + (int64_t)(r0 + r) * A.slices;
        float m = -INFINITY;
        int at = INT32_MAX;
        double sum = 0.0;
        for (int i = lane; i < A.slices; i += 64) {
            const Part p = part[i];
            if (p.m > m || (p.m == m && p.at < at)) {
                if (!GREEDY) sum *= m == -INFINITY ? 0.0 : weight(m, p.m, A.heat);
                m = p.m, at = p.at;
            }
            sum += p.m == -INFINITY || GREEDY ? p.z : p.z * weight(p.m, m, A.heat);
        }
        const float M = wave_max(m);
        if (GREEDY) at = wave_min(m == M ? at : INT32_MAX);
        sum = wave_sum64(m == -INFINITY || GREEDY ? sum : sum * weight(m, M, A.heat));
        if (lane == 0) top[r] = M, z[r] = sum, arg[r] = sum != sum || M == -INFINITY ? -1 : at;
    }
    __syncthreads();
    if (t < n) {
        const int p = par[t], c = tok[t];
        double w = 0.0;
        float d = 0.f;
        if (!GREEDY && p >= 0 && c >= 0 && c < A.V) {
            w = weight(A.x[(int64_t)(r0 + p) * A.ld + c], top[p], A.heat);
            if (A.q) d = A.q[(int64_t)(r0 + p) * A.ldq + c];
        }
        e[t] = w;
        qc[t] = d;
    }
    __syncthreads();
    int cur = 0, n_gone = 0, n_kept = 1;
    double alpha = 0.0, left = 1.0, off = 0.0;
    // The current row's probabilities without what refused drafts took: of one token, and of a range by waves.
    auto rest = [&](int64_t i) -> double {
        const double w = weight(A.x[(int64_t)(r0 + cur) * A.ld + i], top[cur], A.heat);
        if (A.q) {
            const double d = w / z[cur] - alpha * (double)A.q[(int64_t)(r0 + cur) * A.ldq + i];
            return d > 0.0 ? d : 0.0;
        }
        for (int k = 0; k < n_gone; ++k)
            if (gone[k] == i) return 0.0;
        return w;
    };
    // Sums of the pieces of [a, b), one a wave, `len` tokens each, into `piece`.
    auto pieces = [&](int64_t a, int64_t b, int64_t len) {
        double v = 0.0;
        const int64_t from = a + wave * len, to = min(from + len, b);
        for (int64_t i = from + lane; i < to; i += 64) v += rest(i);
        v = wave_sum64(v);
        __syncthreads();
        if (lane == 0) piece[wave] = v;
        __syncthreads();
    };
    auto total = [&]() {
        double v = 0.0;
        for (int w = 0; w < kWalkWaves; ++w) v += piece[w];
        return v;
    };
    const int64_t whole = (A.V + kWalkWaves - 1) / kWalkWaves;
    bool stale = false;   // `left` is of an earlier alpha
    for (int i = 1; i < n; ++i) {
        if (par[i] != cur || tok[i] < 0 || tok[i] >= A.V) continue;
        bool yes;
        if (GREEDY) {
            yes = tok[i] == arg[cur] && arg[cur] >= 0;
        } else if (A.q) {
            if (stale) {
                pieces(0, A.V, whole);
                left = total();
                stale = false;
            }
            const double d = e[i] / z[cur] - alpha * (double)qc[i];
            yes = (double)u[i] * (double)qc[i] * left < (d > 0.0 ? d : 0.0);
            if (!yes) {
                alpha += left;
                stale = true;
            }
        } else {
            bool again = false;   // (the same token twice)
            for (int k = 0; k < n_gone; ++k) again |= gone[k] == tok[i];
            yes = !again && (double)u[i] * (z[cur] - off) < e[i];
            if (!yes && !again) {
                off += e[i];
                __syncthreads();
                if (t == 0) gone[n_gone] = tok[i];
                __syncthreads();
                ++n_gone;
            }
        }
        if (yes) {
            if (t == 0) kept[n_kept] = i;
            ++n_kept;
            cur = i;
            n_gone = 0;
            alpha = off = 0.0;
            left = 1.0;
            stale = false;
        }
    }
    if (t == 0) kept[0] = 0, A.n_kept[s] = n_kept;
    if (t >= n_kept && t < A.max_rows) kept[t] = -1;
    if (GREEDY) {
        if (t == 0) A.next[s] = arg[cur];
        return;
    }
    if (!(z[cur] > 0.0)) {   // (NaN too)
        if (t == 0) A.next[s] = -1;
        return;
    }
    // the first token at which the running sum passes the draw: ever smaller pieces
    int64_t a = 0, b = A.V;
    double want = -1.0;
    for (;;) {
        const int64_t len = (b - a + kWalkWaves - 1) / kWalkWaves;
        pieces(a, b, len);
        double sum = total();
        if (want < 0.0) {
            if (!(sum > 0.0)) {   // nothing left but rounding: the row's own
                alpha = 0.0;
                n_gone = 0;
                pieces(a, b, len);
                sum = total();
            }
            want = (double)u[0] * sum;
        }
        int w = 0, last = 0;
        double before = 0.0, run = 0.0;
        bool found = false;
        for (int k = 0; k < kWalkWaves && !found; ++k) {
            if (piece[k] > 0.0) last = k, before = run;
            run += piece[k];
            found = run > want && piece[k] > 0.0;
        }
        w = last;
        want -= before;
        a += w * len;
        b = min(a + len, b);
        if (b - a <= 64) break;
    }
    if (wave == 0) {
        const double v = a + lane < b ? rest(a + lane) : 0.0;
        double run = v;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const double p = __shfl_up(run, o, 64);
            if (lane >= o) run += p;
        }
        const uint64_t some = __ballot(v > 0.0), past = __ballot(v > 0.0 && run > want);
        if (lane == 0) pick = past ? __builtin_ctzll(past) : some ? 63 - __builtin_clzll(some) : 0;
        if (lane == 0) A.next[s] = (int32_t)(a + pick);
    }
}

// Slices of a row: enough blocks to fill the chip, of at least 1024 tokens.
struct Cut {
    int slices;
    int64_t slice;
};
Cut cut(int n, int64_t V) {
    const int64_t most = std::min<int64_t>(kMaxSlices, (V + 1023) / 1024), want = std::max<int64_t>(1, std::min<int64_t>(most, 2048 / std::max(n, 1)));
    const int64_t slice = ((V + want - 1) / want + 1023) / 1024 * 1024;
    return Cut{(int)((V + slice - 1) / slice), slice};
}

uint64_t ws_bytes_for(uint64_t n_rows, int64_t V) { return std::max<uint64_t>(n_rows, 1) * std::min<int64_t>(kMaxSlices, (V + 1023) / 1024) * sizeof(Part); }

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
    *bytes = ws_bytes_for(n_rows, V);
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
    const uint64_t n = (uint64_t)d->n_rows, ns = (uint64_t)d->n_seqs, need = ws_bytes_for(n, d->vocab);
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
    const Cut c = cut(d->n_rows, d->vocab);
    VfArgs A{d->logits, q ? d->q : nullptr, d->u, d->row0, d->parent, d->token, n_kept, kept, next, (Part *)ws, nullptr, d->ld, d->ldq, d->vocab,
             c.slice, greedy ? 0.0 : 1.0 / (double)d->temp, d->n_seqs, d->n_rows, d->max_rows, c.slices};
    MH_TRY(verify_flag(&A.err));
    for (int r = 0; r < d->n_rows; r += 32768) {   // (a grid's second axis ends at 65535)
        const int k = std::min(32768, d->n_rows - r);
        if (greedy) MH_LAUNCH("verify_part", k_vf_part<true>, dim3((unsigned)c.slices, (unsigned)k), dim3(kThreads), 0, stream(), A, r);
        else MH_LAUNCH("verify_part", k_vf_part<false>, dim3((unsigned)c.slices, (unsigned)k), dim3(kThreads), 0, stream(), A, r);
    }
    if (greedy) MH_LAUNCH("verify_walk", k_vf_walk<true>, dim3((unsigned)d->n_seqs), dim3(kWalk), 0, stream(), A);
    else MH_LAUNCH("verify_walk", k_vf_walk<false>, dim3((unsigned)d->n_seqs), dim3(kWalk), 0, stream(), A);
    return hip_check(hipGetLastError(), "verify launch");
}

}  // extern "C"
