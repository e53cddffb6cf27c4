// kv_q4.cuh -- addressing and checks of the paged 4-bit KV cache (acb_kv_q4), shared by the kernels that
// write it (k_kv_q4.cu) and read it (k_attn_q4.cu).
#pragma once

#include "common.cuh"

namespace acb {

// The format's limit of a scale, so of 8 * 2720 = 21760 for an element. f16 holds (code - 8) d up to d = 8160; the limit is part
// of the format.
constexpr float kQ4MaxScale = 2720.0f;

struct KvQ4 {
    uint8_t *       kc;
    uint16_t *      ks;
    uint8_t *       vc;
    uint16_t *      vs;
    const int32_t * table;
    int64_t         table_stride;
    int             n_pages, page, shift;  // page = 1 << shift tokens
    int             nkv, n_seq, max_pages;

    // page that holds position p of sequence s (s and p in range), -1 outside the pool
    __device__ __forceinline__ int page_of(int s, int p) const {
        const int pg = __ldg(table + (int64_t) s * table_stride + (p >> shift));
        return (unsigned) pg < (unsigned) n_pages ? pg : -1;
    }
    // row number of (page, kv head, slot) in units of one head's token row: below 2^32 (kv_q4_check)
    __device__ __forceinline__ uint32_t row(int pg, int h, int p) const {
        return (((uint32_t) pg * (uint32_t) nkv + (uint32_t) h) << shift) + (uint32_t) (p & (page - 1));
    }
};

inline bool kv_q4_aligned(const void * p) {
    return p && reinterpret_cast<uintptr_t>(p) % 16 == 0;
}

// the status of a caller's cache description, and the device copy of it
inline acb_status kv_q4_check(const acb_kv_q4 * kv, KvQ4 * out) {
    if (!kv || !kv_q4_aligned(kv->k_codes) || !kv_q4_aligned(kv->k_scales) || !kv_q4_aligned(kv->v_codes) ||
        !kv_q4_aligned(kv->v_scales) || !kv->page_table || kv->n_pages <= 0 || kv->n_kv_heads <= 0 || kv->n_seq <= 0 ||
        kv->max_pages <= 0 || kv->table_stride < kv->max_pages || kv->page_size <= 0) {
        return ACB_ERR_INVALID_ARG;
    }
    if ((kv->head_dim != 64 && kv->head_dim != 128 && kv->head_dim != 256) || kv->page_size < 16 ||
        kv->page_size > 4096 || (kv->page_size & (kv->page_size - 1)) != 0 ||
        (int64_t) kv->max_pages * kv->page_size > (1 << 30) ||
        (int64_t) kv->n_pages * kv->n_kv_heads > (int64_t) UINT32_MAX / kv->page_size) {
        return ACB_ERR_UNSUPPORTED;
    }
    int shift = 0;
    while ((1 << shift) < kv->page_size) {
        shift++;
    }
    *out = { kv->k_codes,      kv->k_scales, kv->v_codes,       kv->v_scales, kv->page_table,
             kv->table_stride, kv->n_pages,  kv->page_size,     shift,        kv->n_kv_heads,
             kv->n_seq,        kv->max_pages };
    return ACB_OK;
}

}  // namespace acb
