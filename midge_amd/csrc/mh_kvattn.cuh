// mh_kvattn.cuh — what the two attention kernels over a paged k/v cache share:
// fragments of f16 or MXFP4 rows as f16 matrix operands, two-term f16
// splits, and the arithmetic of the running softmax.
#pragma once

#include <math.h>

#include "mh_kvtree.cuh"

#define KV_INLINE __attribute__((always_inline))

namespace mh {

struct KvAttnArgs {
    KvCacheDev c;
    KvBatchDev b;
    const float *q, *sink;
    float *out, *part;
    unsigned *err;
    int nh, group, window, grid;   // grid: blocks that share the work
    float qscale;                  // scale * log2(e)
    const int32_t *parent;         // trees: of each row (mh_kv_tree_attention_dev)
};

// Columns (rows x heads of a group) of a sequence and k/v head up to which
// the kernel that streams the cache once runs (mh_kvfew.cuh); beyond, the
// one on tiles of 128 columns (mh_kvmany.cuh). 4 k/v heads of 128, the two
// kernels in us for 10 sequences of 2000 tokens, 1 of 8000, 32 of 4000:
// 40 columns f16 40/42, 24/49, 83/79; MXFP4 32/37, 24/46, 62/69; 64 columns
// MXFP4 39/42, 28/47, 73/75, and of 64 41/33, 27/34, 89/81 (8 heads). f16 rows
// past 128, which each wave would load for 16 columns only: 64 columns on 2
// heads of 256 51/52, 36/41, 139/92, 32 columns 42/47, 30/36, 79/88.
inline int kv_few(int dt, int hd) { return dt == MH_KV_F16 && hd > 128 ? 32 : 48; }
// The largest sequence's columns, as the host knows them.
inline int64_t kv_columns(const mh_kv_batch &b, int group) { return (int64_t)(b.row0 ? std::min(b.max_rows, std::max(b.n_rows, 1)) : 1) * group; }
// Trees of up to 64 columns (8 rows of 8 heads) of up to 4 sequences stay with
// the first kernel: the other's three launches and its blocks' starts are most
// of its time. 64 columns on 8 k/v heads, a call of the two in us:
//                1 sequence of 1000   4100   131071    4 of 2000  16000   8 of 2000  32 of 4000
//   MXFP4 of 32               13/20   17/24   52/65       24/24   40/45       32/29       93/63
//            64               14/23   20/28   66/79       27/28   46/52       33/33       90/78
//            96               17/27   28/29  139/120      34/38   83/74       43/40      159/118
//           128               17/27   28/31  105/120      28/40   65/74       37/41      125/120
//   f16   of 32               13/20   16/24   47/63       21/24   36/43       27/28       88/62
//            64               15/24   22/28   77/87       26/28   49/54       31/31      105/87
//            96               19/26   28/28  111/122      32/34   57/67       38/35      132/120
//           128               21/29   26/32  156/153      32/37   84/86       41/40      168/153
// (With many sequences the first kernel's join takes a block a column. Long
// caches of MXFP4 of 96 lose by the rule; the host does not know the lengths.)
inline bool kv_is_few(const mh_kv_cache &c, const mh_kv_batch &b, int group, bool tree) {
    const int64_t columns = kv_columns(b, group);
    return columns <= kv_few(c.dt, c.head_dim) || (tree && columns <= 64 && b.n_seqs <= 4 && c.head_dim <= 128);
}
// The two kernels' workspaces and launches (`tree`: with A.parent), and what
// the entry points check and resolve (mh_kvattn.hip).
uint64_t kv_few_ws(const mh_kv_cache &c, const mh_kv_batch &b, int group);
int kv_few_run(const mh_kv_cache &c, const mh_kv_batch &b, KvAttnArgs A, void *ws);
int kv_few_tree_run(const mh_kv_cache &c, const mh_kv_batch &b, KvAttnArgs A, void *ws);
uint64_t kv_many_ws(const mh_kv_cache &c, const mh_kv_batch &b, int group);
int kv_many_run(const mh_kv_cache &c, const mh_kv_batch &b, KvAttnArgs A, void *ws);
int kv_many_tree_run(const mh_kv_cache &c, const mh_kv_batch &b, KvAttnArgs A, void *ws);

namespace {

typedef _Float16 kv_h2 __attribute__((ext_vector_type(2)));
typedef _Float16 kv_h4 __attribute__((ext_vector_type(4)));
typedef _Float16 kv_h8 __attribute__((ext_vector_type(8)));
typedef float kv_f4 __attribute__((ext_vector_type(4)));
typedef short kv_s4 __attribute__((ext_vector_type(4)));

// A cached row as chunks of CH elements: lane (t, g) = (lane & 15, lane >> 4)
// of a wave takes chunk 4 i + g of token t, i < NL, so that a load of the
// wave covers whole rows of 16 tokens and every chunk is CH / 8 groups of 8
// consecutive elements, the k of one 16x16x32 matrix operand (q is laid out
// alike, and the order of k does not matter). A chunk is as wide as the row
// allows: 16 bytes, or 8 or 4 where four lanes' share is no more.
template <int DT, int HD>
struct KvRow {
    static constexpr int CH = DT == MH_KV_F16 ? 8 : HD % 128 == 0 ? 32 : HD % 64 == 0 ? 16 : 8;
    static constexpr int NL = HD / (4 * CH);
    static constexpr int BYTES = DT == MH_KV_F16 ? 2 * CH : CH / 2;   // of a chunk
    static constexpr int W = BYTES / 4;                              // dwords
    static constexpr int ROW = DT == MH_KV_F16 ? 2 * HD : HD / 2;    // bytes of a row
    static constexpr int KS = HD / 32;                               // k steps
};

// A lane's raw chunks of one token row.
template <int DT, int HD>
struct KvFrag {
    using R = KvRow<DT, HD>;
    uint32_t w[R::NL][R::W];
    uint32_t e[DT == MH_KV_F16 ? 1 : R::NL];   // exponent bytes

    // rows: the first of 16 token rows, exps: their exponent bytes (the same for
    // the wave, so that the loads take them as scalars); off, eoff: lane_off()
    __device__ __forceinline__ void load(const uint8_t *rows, const uint8_t *exps, uint32_t off, uint32_t eoff) {
#pragma unroll
        for (int i = 0; i < R::NL; ++i) {
            mh_gbytes p = mh_global(rows) + 4 * i * R::BYTES + off;
            if constexpr (R::W == 4) {
                const mh_u4 v = mh_load16_cached(p);
                w[i][0] = v.x;
                w[i][1] = v.y;
                w[i][2] = v.z;
                w[i][3] = v.w;
            } else if constexpr (R::W == 2) {
                const uint64_t v = *(const uint64_t __attribute__((address_space(1))) *)p;
                w[i][0] = (uint32_t)v;
                w[i][1] = (uint32_t)(v >> 32);
            } else {
                w[i][0] = *(const uint32_t __attribute__((address_space(1))) *)p;
            }
            if constexpr (DT != MH_KV_F16) e[i] = *(mh_global(exps) + 4 * i * R::CH / 32 + eoff);
        }
    }
    // where lane (t, g)'s first chunk and its exponent byte are
    static __device__ __forceinline__ uint32_t lane_off(int t, int g) { return (uint32_t)(t * R::ROW + g * R::BYTES); }
    static __device__ __forceinline__ uint32_t lane_eoff(int t, int g) { return (uint32_t)(t * (HD / 32) + g * R::CH / 32); }
    __device__ __forceinline__ void zero() {
#pragma unroll
        for (int i = 0; i < R::NL; ++i) {
#pragma unroll
            for (int j = 0; j < R::W; ++j) w[i][j] = 0u;
            if constexpr (DT != MH_KV_F16) e[i] = 127u;
        }
    }
    // elements 8 s .. 8 s + 7 of chunk i
    __device__ __forceinline__ kv_h8 eight(int i, int s) const {
        kv_h8 r;
        if constexpr (DT == MH_KV_F16) {
            __builtin_memcpy(&r, &w[i][0], 16);
        } else {
            const float sc = __uint_as_float(e[i] << 23);   // 2^(byte - 127); byte 255 makes the converter give NaN
            const kv_h2 a = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w[i][s], sc, 0);
            const kv_h2 b = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w[i][s], sc, 1);
            const kv_h2 c = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w[i][s], sc, 2);
            const kv_h2 d = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w[i][s], sc, 3);
            r = kv_h8{a.x, a.y, b.x, b.y, c.x, c.y, d.x, d.y};
        }
        return r;
    }
};

// A word of the batch's or the plan's arrays, which no kernel that reads it
// so writes: a scalar load where the index is the wave's.
__device__ __forceinline__ int32_t kv_word(const int32_t *p, int64_t i) {
    return ((const int32_t __attribute__((address_space(4))) *)p)[i];
}

// Whether a column whose row is at position pos sees token tok: 0 <= pos - tok
// < w; of a tree's own tokens, from base on, those on the row's path. `rarely`
// is the same from the window itself, for a path that few calls take: no bound
// made of it then holds a register in every tile (of MXFP4 of 256, 17 to 32
// columns, the tiles' loads come in another order then: 16 sequences of 3000
// tokens, 4 k/v heads, 54 us for 48).
template <bool TREE>
struct KvSees {
    __device__ __forceinline__ bool operator()(int pos, int, int tok, uint32_t w) const { return (uint32_t)(pos - tok) < w; }
    __device__ __forceinline__ bool rarely(int pos, int, int tok, int window) const { return tok <= pos && (window <= 0 || tok > pos - window); }
};
template <>
struct KvSees<true> {
    uint64_t path = 0;
    __device__ __forceinline__ bool operator()(int pos, int base, int tok, uint32_t w) const {
        const uint32_t i = (uint32_t)(tok - base);
        return i < (uint32_t)kTreeRows ? path >> i & 1 : (uint32_t)(pos - tok) < w;
    }
    __device__ __forceinline__ bool rarely(int pos, int base, int tok, int window) const {
        const uint32_t i = (uint32_t)(tok - base);
        return i < (uint32_t)kTreeRows ? path >> i & 1 : tok <= pos && (window <= 0 || tok > pos - window);
    }
};

// The position of row `row` of a sequence (-1: no row, or padding) and what
// it sees; paths as kv_paths gives them. Called by whole waves.
template <bool TREE>
__device__ __forceinline__ int kv_column(const KvAttnArgs &A, const KvSeq &q, uint64_t paths, int row, KvSees<TREE> *sees) {
    if constexpr (TREE) {
        const unsigned long long s = __shfl((unsigned long long)paths, max(row, 0), 64);
        sees->path = row < 0 ? 0ull : A.window > 0 ? kv_nearest(s, A.window) : s;
        return row < 0 ? -1 : q.len - q.n + __popcll(s) - 1;
    } else {
        return row < 0 ? -1 : max(q.len - q.n + row, -1);
    }
}

// Any element of eight that is inf or NaN.
__device__ __forceinline__ bool kv_odd(kv_h8 v) {
    uint32_t w[4];
    __builtin_memcpy(w, &v, 16);
    bool r = false;
#pragma unroll
    for (int i = 0; i < 4; ++i) r |= (w[i] & 0x7c00u) == 0x7c00u || (w[i] & 0x7c000000u) == 0x7c000000u;
    return r;
}

// x as two f16 terms: x = hi + lo up to 2^-22 of x (for x within f16's normal
// range by the callers' scaling).
__device__ __forceinline__ void kv_split(float x, _Float16 *hi, _Float16 *lo) {
    *hi = (_Float16)x;
    *lo = (_Float16)(x - (float)*hi);
}

// Two at once: the first terms rounded toward zero by one instruction (the
// second ones take up what that leaves), the second ones to nearest. `minus`
// is -1 that the compiler does not know, so that it keeps the fused
// multiply-add which reads and writes f16 (a subtraction would take a
// conversion on either side).
__device__ __forceinline__ float kv_minus() {
    float m = -1.f;
    asm volatile("" : "+s"(m));
    return m;
}
__device__ __forceinline__ void kv_split2(float x, float y, float minus, kv_h2 *hi, kv_h2 *lo) {
    const auto h = __builtin_amdgcn_cvt_pkrtz(x, y);
    __builtin_memcpy(hi, &h, 4);
    *lo = kv_h2{(_Float16)__builtin_fmaf((float)(*hi)[0], minus, x), (_Float16)__builtin_fmaf((float)(*hi)[1], minus, y)};
}

// A weight is 2^(s - m + kBias) with s - m <= kLag (the running maximum m is
// only moved when a score passes it by more): at most 2^15, the first f16 term
// normal down to 2^-23 of the largest, the second down to 2^-12 and then off by
// at most half a subnormal's step, 2^-34 of the largest.
constexpr float kBias = 9.f, kLag = 6.f;

// floor(a / b) for 0 <= a < 2^52, 0 < b: the quotient's rounding stays below
// the distance to the next whole number (and 64-bit integers are divided in
// some 130 instructions).
__device__ __forceinline__ int64_t kv_div(int64_t a, int64_t b) { return (int64_t)((double)a / (double)b); }

// v of lane ^ 8 within rows of 16 (row_ror:8)
__device__ __forceinline__ float kv_ror8(float v) {
    return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x128, 0xF, 0xF, false));
}

// One wave's tr16 read: 4 rows of 16 f16 as columns (lane i of 16 gives the
// address of 4 elements of row i / 4 and gets column i of the four rows).
__device__ __forceinline__ kv_h4 kv_tr16(const _Float16 *p) {
    const kv_s4 v = __builtin_amdgcn_ds_read_tr16_b64_v4i16((kv_s4 __attribute__((address_space(3))) *)p);
    kv_h4 r;
    __builtin_memcpy(&r, &v, 8);
    return r;
}

}  // namespace
}  // namespace mh
