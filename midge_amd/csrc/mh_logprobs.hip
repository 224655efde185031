// mh_logprobs.hip — log probabilities of given tokens, the entropy and the
// most probable tokens of rows of logits (mh_logprobs_dev).
#include <math.h>

#include "mh_internal.h"

namespace mh {
namespace {

constexpr int kLpTop = 64;

struct LpArgs {
    const float *x;
    const int32_t *ids;
    float *lp, *entropy, *top_lp;
    int32_t *top_id;
    int64_t ld, V;
    int m, top;
};

__device__ __forceinline__ float block_max(float v, float *red) {
    for (int j = 32; j; j >>= 1) v = fmaxf(v, __shfl_xor(v, j, 64));
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    return fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
}
__device__ __forceinline__ float block_sum(float v, float *red) {
    for (int j = 32; j; j >>= 1) v += __shfl_xor(v, j, 64);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    return red[0] + red[1] + red[2] + red[3];
}

// A key that orders as the alternatives do: larger logits first, then lower
// ids; NaNs behind everything.
__device__ __forceinline__ uint64_t order_key(float x, uint32_t id) {
    uint32_t u = __float_as_uint(x == 0.f ? 0.f : x);   // -0 ranks as 0
    u = u >> 31 ? ~u : u | 0x80000000u;
    if (x != x) u = 0;
    return (uint64_t)u << 32 | (uint32_t)~id;
}

// One block a row.
__global__ void __launch_bounds__(256) k_logprobs(LpArgs A) {
    __shared__ float red[4];
    __shared__ uint64_t kred[4];
    const float *x = A.x + (int64_t)blockIdx.x * A.ld;
    const int t = threadIdx.x;
    float m = -INFINITY;
    bool bad = false;
    for (int64_t i = t; i < A.V; i += 256) {
        m = fmaxf(m, x[i]);
        bad |= x[i] != x[i];
    }
    m = block_max(m, red);
    bad = __syncthreads_or(bad || m == INFINITY);
    const bool none = m == -INFINITY;
    float z = 0.f, w = 0.f;
    for (int64_t i = t; i < A.V; i += 256) {
        const float d = x[i] - m, e = expf(d);
        z += e;
        w += e > 0.f ? e * d : 0.f;
    }
    z = block_sum(z, red);
    w = block_sum(w, red);
    const float lz = logf(z);
    auto lp = [&](float v) { return bad ? NAN : none ? -INFINITY : (v - m) - lz; };
    for (int j = t; j < A.m; j += 256) {
        const int id = A.ids[(int64_t)blockIdx.x * A.m + j];
        A.lp[(int64_t)blockIdx.x * A.m + j] = id >= 0 && id < A.V ? lp(x[id]) : bad ? NAN : -INFINITY;
    }
    if (t == 0 && A.entropy) A.entropy[blockIdx.x] = bad ? NAN : none ? 0.f : lz - w / z;
    uint64_t last = ~0ull;
    for (int j = 0; j < A.top; ++j) {
        uint64_t best = 0;
        for (int64_t i = t; i < A.V; i += 256) {
            const uint64_t k = order_key(x[i], (uint32_t)i);
            if (k < last && k > best) best = k;
        }
        for (int o = 32; o; o >>= 1) {
            const uint64_t k = __shfl_xor((unsigned long long)best, o, 64);
            best = k > best ? k : best;
        }
        __syncthreads();
        if ((t & 63) == 0) kred[t >> 6] = best;
        __syncthreads();
        for (int o = 0; o < 4; ++o) best = kred[o] > best ? kred[o] : best;
        last = best;
        if (t == 0) {
            const uint32_t id = ~(uint32_t)best;
            A.top_id[(int64_t)blockIdx.x * A.top + j] = (int32_t)id;
            A.top_lp[(int64_t)blockIdx.x * A.top + j] = lp(x[id]);
        }
    }
}

int validate(int n, int64_t V, int top, const char *what) {
    if (n < 0 || n > (1 << 24)) return fail(MH_E_ARG, "%s: %d rows", what, n);
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
    *bytes = 16;
    return MH_OK;
}

int mh_logprobs_dev(const float *logits, int64_t ld, int n, int64_t V, const int32_t *ids, int m, int top, float *lp,
                    float *entropy, int32_t *top_id, float *top_lp, void *ws, uint64_t ws_bytes) {
    const char *what = "mh_logprobs_dev";
    uint64_t need = 0;
    clear_error();
    MH_TRY(validate(n, V, top, what));
    MH_TRY(mh_logprobs_ws(n, V, top, &need));
    if (!logits || !ws) return fail(MH_E_ARG, "%s: NULL logits or workspace", what);
    if (ld < V || ld > ((int64_t)1 << 40)) return fail(MH_E_ARG, "%s: rows of %lld floats, %lld tokens", what, (long long)ld, (long long)V);
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
    MH_TRY(resolve_here(logits, 4 * ((uint64_t)(n - 1) * ld + V), what));
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
    LpArgs A{logits, ids, lp, entropy, top_lp, top_id, ld, V, m, top};
    MH_LAUNCH("logprobs", k_logprobs, dim3((unsigned)n), dim3(256), 0, stream(), A);
    return hip_check(hipGetLastError(), "logprobs launch");
}

}  // extern "C"
