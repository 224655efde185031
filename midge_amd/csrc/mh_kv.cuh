// mh_kv.cuh — paged k/v caches: the descriptors as the kernels see them, the
// bounds that device-held batch data is checked against (shared with the
// host-side mh_kv_check), and the MXFP4 block encoding.
#pragma once

#include "mh_internal.h"

namespace mh {

struct KvCacheDev {
    uint8_t *k, *v, *ks, *vs;
    int64_t n_pages;
    int dt, nkv, hd, shift;   // page = 1 << shift tokens
};

struct KvBatchDev {
    const int32_t *row0, *len, *pages;
    int n_seqs, n_rows, max_rows, max_pages;
};

// A sequence's rows [r0, r0 + n) and length.
struct KvSeq {
    int r0, n, len;
};

// What sequence s of a batch is, false if its rows or length are out of
// bounds (nothing of it is then followed).
__host__ __device__ inline bool kv_seq(const KvBatchDev &b, int shift, int s, KvSeq *q) {
    const int r0 = b.row0 ? b.row0[s] : s, r1 = b.row0 ? b.row0[s + 1] : s + 1;
    const int len = b.len[s];
    q->r0 = r0;
    q->n = r1 - r0;
    q->len = len;
    return r0 >= 0 && r1 >= r0 && r1 <= b.n_rows && r1 - r0 <= b.max_rows && len >= 0 &&
           (int64_t)len <= ((int64_t)b.max_pages << shift);
}

// Page number valid?
__host__ __device__ inline bool kv_page_ok(const KvCacheDev &c, int page) {
    return page >= 0 && (int64_t)page < c.n_pages;
}

// Index of the token row (head_dim elements) of a slot of a page.
__host__ __device__ inline uint64_t kv_slot(const KvCacheDev &c, int page, int head, int slot) {
    return ((((uint64_t)page * (unsigned)c.nkv + (unsigned)head) << c.shift) + (unsigned)slot);
}

// Host side (mh_kv.hip): argument checks without a device, then resolution.
int kv_validate(const mh_kv_cache *c, const mh_kv_batch *b, const char *what);
int kv_resolve(const mh_kv_cache *c, const mh_kv_batch *b, KvCacheDev *cd, KvBatchDev *bd, const char *what);
// Memory that the call writes, apart from the cache's and the batch's.
int kv_apart(const mh_kv_cache *c, const mh_kv_batch *b, const void *p, uint64_t bytes, const char *what);
// Ranges of bytes that share an address.
inline bool kv_overlap(const void *a, uint64_t na, const void *b, uint64_t nb) {
    return (uintptr_t)a < (uintptr_t)b + nb && (uintptr_t)b < (uintptr_t)a + na;
}

// The exponent byte of an MXFP4 block whose largest magnitude has the f32
// bits `top` (sign cleared): the smallest e in [-13, 13] with amax <= 7 * 2^e,
// plus 127; 255 if it is not finite. amax = f * 2^x, f in [0.5, 1): e = x - 3
// where f <= 7/8 (mantissa field <= 0x600000), else x - 2.
__host__ __device__ inline int kv_block_exp(uint32_t top) {
    if (top >= 0x7f800000u) return 255;
    int e = (int)(top >> 23) - 126 - 3 + ((top & 0x7fffffu) > 0x600000u);
    e = e < -13 ? -13 : e > 13 ? 13 : e;
    return e + 127;
}

}  // namespace mh
