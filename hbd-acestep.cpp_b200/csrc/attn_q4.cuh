// attn_q4.cuh -- what the two forms of attention over the 4-bit cache share: their arguments, the bounds of a sequence and
// the unpacking of codes (k_attn_q4.cu: few rows, small tensor-core tiles; k_attn_q4_tc.cu: many rows, tcgen05).
#pragma once

#include "kv_q4.cuh"

namespace acb {

struct AttnQ4Args {
    const void *    q;
    int64_t         q_stride, n_tok;
    int             Nh, G;
    const int32_t * q_start;
    const int32_t * kv_len;
    int             max_q, max_kv, window;
    float           scale_log2;
    void *          o;
    int64_t         o_stride;
    int *           err;
    KvQ4            kv;
    bool            q_vec;    // rows of q are 16-byte aligned
    int             chunk;    // keys of a block, a multiple of 64
    int             tiles;    // of the rows
    int             n_split;  // chunks that the rows of one block can touch
    int64_t         rows;     // tokens that sequences can have: n_tok, or max_q of each where that is less
    bool            by_seq;   // parts by sequence and its new token, not by token (max_q of each is less)
    float *         part_o;   // [rows*Nh][n_split][D]: sums of P V
    float2 *        part_ml;  // [rows*Nh][n_split]: m (log2), l
};

// rows and keys of sequence s as the device arrays give them; false when they are outside the call's bounds
__device__ __forceinline__ bool seq_bounds(const AttnQ4Args & a, int s, int64_t * row0, int * n, int * len) {
    const int64_t q0 = a.q_start ? __ldg(a.q_start + s) : s;
    const int64_t q1 = a.q_start ? __ldg(a.q_start + s + 1) : s + 1;
    *len             = __ldg(a.kv_len + s);
    *row0            = q0;
    *n               = (int) min((int64_t) a.max_q, max((int64_t) 0, q1 - q0));
    return q0 >= 0 && q1 >= q0 && q1 <= a.n_tok && q1 - q0 <= a.max_q && *len >= 0 && *len <= a.max_kv;
}

__device__ __forceinline__ uint32_t u32_of(__half2 h) {
    return *reinterpret_cast<uint32_t *>(&h);
}

__device__ __forceinline__ __half2 half2_of(uint32_t u) {
    return *reinterpret_cast<__half2 *>(&u);
}

// The four pairs of codes of a word (low and high nibbles of bytes 0 and 2, then of bytes 1 and 3) times the pair of
// scales. 0x6400 | c is the f16 number 1024 + c and 0x6400 | 16 c is 1024 + 16 c, so that c - 8 comes from one exact f16
// operation; times d is exact by the scales' 8 bits.
__device__ __forceinline__ void unpack4(uint32_t w, __half2 d, uint32_t * r) {
    const __half2  b0 = half2_of(0xE408E408u);  // -1032
    const __half2  sx = half2_of(0x2C002C00u);  // 1/16
    const __half2  b1 = half2_of(0xD480D480u);  // -72
    const uint32_t u  = w >> 8;
    r[0] = u32_of(__hmul2(__hadd2(half2_of((w & 0x000F000Fu) | 0x64006400u), b0), d));
    r[1] = u32_of(__hmul2(__hfma2(half2_of((w & 0x00F000F0u) | 0x64006400u), sx, b1), d));
    r[2] = u32_of(__hmul2(__hadd2(half2_of((u & 0x000F000Fu) | 0x64006400u), b0), d));
    r[3] = u32_of(__hmul2(__hfma2(half2_of((u & 0x00F000F0u) | 0x64006400u), sx, b1), d));
}

template <int N> struct Words {
    uint32_t w[N];
    template <class Load> __device__ __forceinline__ void load_with(const void * p, Load ld) {
        if constexpr (N % 4 == 0) {
#pragma unroll
            for (int i = 0; i < N / 4; i++) {
                const uint4 u = ld(reinterpret_cast<const uint4 *>(p) + i);
                w[4 * i] = u.x, w[4 * i + 1] = u.y, w[4 * i + 2] = u.z, w[4 * i + 3] = u.w;
            }
        } else if constexpr (N == 2) {
            const uint2 u = ld(reinterpret_cast<const uint2 *>(p));
            w[0] = u.x, w[1] = u.y;
        } else {
            w[0] = ld(reinterpret_cast<const uint32_t *>(p));
        }
    }
    __device__ __forceinline__ void load(const void * p) {
        load_with(p, [](auto * q) { return __ldg(q); });
    }
    __device__ __forceinline__ void load_shared(const void * p) {
        load_with(p, [](auto * q) { return *q; });
    }
};

// many rows per sequence and kv head (16-bit q and o, heads of 64 and 128); false where the call is not one for it
bool attn_q4_tc_wanted(const AttnQ4Args & a, int type, int head_dim);
acb_status attn_q4_tc_launch(const AttnQ4Args & a, int type, int head_dim, cudaStream_t st);

}  // namespace acb
