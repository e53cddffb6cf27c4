// k_kv_q4.cu -- the writes of the paged 4-bit KV cache (acb_kv_q4_append: norm, rotation, quantisation and scatter in
// one pass over the fused qkv rows) and the rows read back as values (acb_kv_q4_read).
//
// A block of 32 values x is held as d (code - 8) with d = f16(bf16(-mx / 8)), mx the value of largest magnitude: mx itself
// gets code 0, its negative side reaches 15. Rounding d to bf16 (8 significant bits; 2^-9 of the block's largest value
// against the codes' own step of 2^-4) makes every product d (code - 8) an f16 number, because |code - 8| <= 8 has at most
// 3 significant bits: the attention's operands are then exact. The codes come from a correctly rounded division, so that a
// quotient that is exactly between two codes (16-bit inputs often are) goes the same way everywhere.
//
// The bytes of q, k and v bound it. The fast form: a block per token, a thread 8 consecutive elements of a head, so that a
// block of 32 is four lanes, a rotation's partner is in the thread (interleaved) or another lane's (half), and the angles of
// a thread's elements serve every head that it takes. Rows that are not 16-byte aligned, or rotated widths that do not fall on
// vectors, go a warp to a head through shared memory. 17002 tokens of 16 + 8 + 8 heads of 128, bf16, normed and rotated: 89 us,
// 2.4 TB/s of 217 MB, and 23 us for reading the rows back as f16 (4.7 TB/s of 109 MB). Both together 112 us; a warp to a head
// 330, codes by a division each 205, one loop over rows of all kinds 167, four warps to every token 126, four rows a thread in
// flight instead of two 136 (one: 116), room for 28 warps an SM 114 (the rotation spills), for 20 116. 1100
// instructions for the four rows of a warp hold the append there: the codes are 100 a row, the norm's sum in double 60, the
// rotation's exchange 50.
#include <algorithm>

#include "kv_q4.cuh"

namespace acb {
namespace {

struct AppendArgs {
    const void *    qkv;
    int64_t         stride, n_tok;
    int             Nh;
    const float *   q_norm;
    const float *   k_norm;
    float           eps;
    const float *   table;
    int             max_pos, R;
    bool            half;
    const int32_t * seq;
    const int32_t * pos;
    void *          q_out;
    int64_t         q_stride;
    int *           err;
    KvQ4            kv;
};

__device__ __forceinline__ float max_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}

__device__ __forceinline__ float min_nan(float a, float b) {
    float r;
    asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}

// the scale of a block from its largest and smallest value
__device__ __forceinline__ __half q4_scale(float hi, float lo) {
    const float mx = hi >= -lo ? hi : lo;
    float       d  = __fmul_rn(mx, -0.125f);
    if (d == d) {
        d = fminf(fmaxf(d, -kQ4MaxScale), kQ4MaxScale);
    }
    return __float2half_rn(__bfloat162float(__float2bfloat16_rn(d)));
}

__device__ __forceinline__ uint32_t q4_code(float x, float d) {
    return d == 0.0f ? 8u : (uint32_t) fminf(fmaxf(floorf(__fadd_rn(__fdiv_rn(x, d), 8.5f)), 0.0f), 15.0f);
}

// The codes of 4 values, a byte each, without a division. m = rint(x * (1/d) + 8.5) is the border nearest to x / d + 8.5, and
// (m - 8.5) d has 13 bits, so e = x - (m - 8.5) d is exact next to the border: on it (as 16-bit inputs often are) or
// at least 2^-18 d off, its sign says on which side the division falls. *near is the smallest distance that is neither, as the
// bits of a float less one. y is held between the borders 0 | 1 and 15; a NaN scale gives some code.
__device__ __forceinline__ uint32_t q4_codes4(const float * x, float d, float inv, uint32_t * near) {
    const float off = __fmul_rn(d, -8.5f);
    uint32_t    c   = 0;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const float y = fminf(fmaxf(__fmaf_rn(x[i], inv, 8.5f), 0.75f), 15.25f);
        const float r = __fadd_rn(y, 8388608.0f);  // 2^23: the bits of the sum are those of 2^23 plus m
        const float m = __fsub_rn(r, 8388608.0f);
        const float e = __fmaf_rn(__fsub_rn(x[i], __fmaf_rn(m, d, off)), inv, 0.0f);  // + 0 makes -0 a 0
        *near         = min(*near, (__float_as_uint(e) & 0x7FFFFFFFu) - 1u);
        c += ((uint32_t) (__float_as_int(r) + (__float_as_int(e) >> 31)) & 15u) << (8 * i);
    }
    return c;
}

// one warp per (token, head of q | k | v); the head's row goes through shared memory, where every pair of every layout
// is at hand
template <int TI, int TQ, int D> __global__ void __launch_bounds__(256) kv_q4_append_kernel(const AppendArgs a) {
    constexpr int     E = D / 32;
    __shared__ float  rows[8][D];
    const int         lane = threadIdx.x & 31;
    float *           x    = rows[threadIdx.x >> 5];
    const int         nh   = a.Nh + 2 * a.kv.nkv;
    const int64_t     item = (int64_t) blockIdx.x * 8 + (threadIdx.x >> 5);
    if (item >= a.n_tok * nh) {
        return;
    }
    const int64_t t = item / nh;
    const int     h = (int) (item - t * nh);
    const int     s = __ldg(a.seq + t), p = __ldg(a.pos + t);
    if (s < 0) {
        return;
    }
    const bool is_q = h < a.Nh, is_v = h >= a.Nh + a.kv.nkv;
    int        bad = s >= a.kv.n_seq ? ACB_DEVERR_ID_RANGE : 0;
    if (p < 0 || (p >> a.kv.shift) >= a.kv.max_pages || (a.table && p >= a.max_pos)) {
        bad |= ACB_DEVERR_POS_RANGE;
    }
    const int pg = bad ? -1 : a.kv.page_of(s, p);
    if (!bad && pg < 0) {
        bad = ACB_DEVERR_PAGE_RANGE;
    }
    typename io<TQ>::t * q = reinterpret_cast<typename io<TQ>::t *>(a.q_out) + t * a.q_stride + (int64_t) h * D;
    if (bad) {
        if (lane == 0 && a.err) {
            atomicOr(a.err, bad);
        }
        if (is_q) {
            for (int e = 0; e < E; e++) {
                q[e * 32 + lane] = io<TQ>::from_f(0.0f);
            }
        }
        return;
    }
    const typename io<TI>::t * src = reinterpret_cast<const typename io<TI>::t *>(a.qkv) + t * a.stride + (int64_t) h * D;
    float                      v[E];
#pragma unroll
    for (int e = 0; e < E; e++) {
        v[e] = io<TI>::to_f(src[e * 32 + lane]);
    }
    if (!is_v) {
        const float * w = is_q ? a.q_norm : a.k_norm;
        if (w) {
            double ss = 0.0;
#pragma unroll
            for (int e = 0; e < E; e++) {
                ss += (double) __fmul_rn(v[e], v[e]);
            }
            const float sc = rms_scale_pow2<D>(warp_sum(ss), a.eps);
#pragma unroll
            for (int e = 0; e < E; e++) {
                v[e] = __fmul_rn(__fmul_rn(v[e], sc), __ldg(w + e * 32 + lane));
            }
        }
        if (a.table) {
#pragma unroll
            for (int e = 0; e < E; e++) {
                x[e * 32 + lane] = v[e];
            }
            __syncwarp();
            const float * w2 = a.table + (int64_t) p * a.R;
            for (int i = lane; i < a.R / 2; i += 32) {
                const int   ia = a.half ? i : 2 * i, ib = a.half ? i + a.R / 2 : 2 * i + 1;
                const float c = __ldg(w2 + 2 * i), sn = __ldg(w2 + 2 * i + 1), u = x[ia], z = x[ib];
                x[ia] = __fsub_rn(__fmul_rn(u, c), __fmul_rn(z, sn));
                x[ib] = __fadd_rn(__fmul_rn(u, sn), __fmul_rn(z, c));
            }
            __syncwarp();
#pragma unroll
            for (int e = 0; e < E; e++) {
                v[e] = x[e * 32 + lane];
            }
        }
    }
    if (is_q) {
#pragma unroll
        for (int e = 0; e < E; e++) {
            q[e * 32 + lane] = io<TQ>::from_f(v[e]);
        }
        return;
    }
    const int64_t row    = a.kv.row(pg, is_v ? h - a.Nh - a.kv.nkv : h - a.Nh, p);
    uint8_t *     codes  = (is_v ? a.kv.vc : a.kv.kc) + row * (D / 2);
    uint16_t *    scales = (is_v ? a.kv.vs : a.kv.ks) + row * E;
#pragma unroll
    for (int e = 0; e < E; e++) {
        float hi = v[e], lo = v[e];
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            hi = max_nan(hi, __shfl_xor_sync(0xffffffffu, hi, o));
            lo = min_nan(lo, __shfl_xor_sync(0xffffffffu, lo, o));
        }
        const __half   d = q4_scale(hi, lo);
        const uint32_t c = q4_code(v[e], __half2float(d));
        const uint32_t u = __shfl_down_sync(0xffffffffu, c, 16);
        if (lane < 16) {
            codes[e * 16 + lane] = (uint8_t) (c | (u << 4));
        }
        if (lane == 0) {
            scales[e] = __half_as_ushort(d);
        }
    }
}

// LPR lanes to a head's row; ROPE 0: none, 1: half pairs, 2: interleaved. The rows of q, k and v are gone through one kind
// after the other, U rows a thread in flight, each kind's first rows loaded before anything else.
constexpr int kAppendWarps = 4;  // of a block at most
constexpr int kAppendRoom  = 24;  // warps of an SM

template <int TI, int TQ, int D, int ROPE>
__global__ void __launch_bounds__(32 * kAppendWarps, kAppendRoom / kAppendWarps) kv_q4_append_vec_kernel(const AppendArgs a) {
    constexpr int LPR = D / 8, RPW = 32 / LPR, VI = vec16<TI>::N, VQ = vec16<TQ>::N, U = TI == ACB_TYPE_F32 ? 1 : 2;
    const int     TURN = (int) (blockDim.x >> 5) * RPW;  // rows of one row a thread
    using EI           = typename io<TI>::t;
    const int64_t t    = blockIdx.x;
    const int     lane = threadIdx.x & 31, sub = lane % LPR, d0 = sub * 8;
    const int     r0   = (threadIdx.x >> 5) * RPW;  // the warp's first row of a turn
    const int     rl   = lane / LPR;                // this lane's row among the warp's
    const int     s = __ldg(a.seq + t), p = __ldg(a.pos + t);
    const EI *    src[3];
    src[0] = reinterpret_cast<const EI *>(a.qkv) + t * a.stride + d0;
    src[1] = src[0] + (int64_t) a.Nh * D;
    src[2] = src[1] + (int64_t) a.kv.nkv * D;
    vec16<TI> in[3][U][8 / VI];
    auto      load = [&](int kind, int r, int n) {
#pragma unroll
        for (int u = 0; u < U; u++) {
            if (r + u * TURN + rl < n) {
#pragma unroll
                for (int i = 0; i < 8 / VI; i++) {
                    in[kind][u][i].load(src[kind] + (r + u * TURN + rl) * D + i * VI);
                }
            }
        }
    };
    load(0, r0, a.Nh);
    load(1, r0, a.kv.nkv);
    load(2, r0, a.kv.nkv);
    if (s < 0) {
        return;
    }
    int bad = s >= a.kv.n_seq ? ACB_DEVERR_ID_RANGE : 0;
    if (p < 0 || (p >> a.kv.shift) >= a.kv.max_pages || (ROPE && p >= a.max_pos)) {
        bad |= ACB_DEVERR_POS_RANGE;
    }
    const int pg = bad ? -1 : a.kv.page_of(s, p);
    if (!bad && pg < 0) {
        bad = ACB_DEVERR_PAGE_RANGE;
    }
    if (bad && threadIdx.x == 0 && a.err) {
        atomicOr(a.err, bad);
    }
    float      c[8], sn[8];  // sn with the sign that its product has in this lane's sum
    const int  half = a.R / 2;
    const bool turn = ROPE && !bad && d0 < a.R;
    // the lane with the other half of this lane's pairs
    const int  mate = ROPE == 1 && d0 < a.R ? lane + (d0 < half ? half / 8 : -(half / 8)) : lane;
    const bool up   = ROPE == 1 && d0 >= half;
    if (turn) {
        const float4 * w = reinterpret_cast<const float4 *>(a.table + (int64_t) p * a.R + (ROPE == 1 ? 2 * (up ? d0 - half : d0) : d0));
#pragma unroll
        for (int e = 0; e < (ROPE == 1 ? 4 : 2); e++) {
            const float4 f = __ldg(w + e);
            c[2 * e] = f.x, sn[2 * e] = f.y, c[2 * e + 1] = f.z, sn[2 * e + 1] = f.w;
        }
        if (ROPE == 1 && !up) {
#pragma unroll
            for (int e = 0; e < 8; e++) {
                sn[e] = -sn[e];
            }
        }
    }
    float ww[8];
    auto  weights = [&](const float * w) {
        const float4 w0 = __ldg(reinterpret_cast<const float4 *>(w + d0)), w1 = __ldg(reinterpret_cast<const float4 *>(w + d0) + 1);
        ww[0] = w0.x, ww[1] = w0.y, ww[2] = w0.z, ww[3] = w0.w, ww[4] = w1.x, ww[5] = w1.y, ww[6] = w1.z, ww[7] = w1.w;
    };
    auto norm_turn = [&](float * x, bool norm) {
        if (norm) {
            double ss = 0.0;
#pragma unroll
            for (int i = 0; i < 8; i++) {
                ss += (double) __fmul_rn(x[i], x[i]);
            }
#pragma unroll
            for (int o = LPR / 2; o > 0; o >>= 1) {
                ss += __shfl_xor_sync(0xffffffffu, ss, o);
            }
            const float sc = rms_scale_pow2<D>(ss, a.eps);
#pragma unroll
            for (int i = 0; i < 8; i++) {
                x[i] = __fmul_rn(__fmul_rn(x[i], sc), ww[i]);
            }
        }
        if (ROPE == 1) {
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const float z = __shfl_sync(0xffffffffu, x[i], mate);
                const float r = __fadd_rn(__fmul_rn(x[i], c[i]), __fmul_rn(z, sn[i]));  // a c - b s, b c + a s
                x[i]          = turn ? r : x[i];
            }
        } else if (ROPE == 2 && turn) {
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const float y = x[2 * i], z = x[2 * i + 1];
                x[2 * i]     = __fsub_rn(__fmul_rn(y, c[i]), __fmul_rn(z, sn[i]));
                x[2 * i + 1] = __fadd_rn(__fmul_rn(y, sn[i]), __fmul_rn(z, c[i]));
            }
        }
    };
    // a row into the cache: blocks of 32 are four lanes
    auto quantise = [&](const float * x, bool live, int h, uint8_t * codes, uint16_t * scales) {
        float hi = x[0], lo = x[0];
#pragma unroll
        for (int i = 1; i < 8; i++) {
            hi = max_nan(hi, x[i]);
            lo = min_nan(lo, x[i]);
        }
#pragma unroll
        for (int o = 1; o <= 2; o <<= 1) {
            hi = max_nan(hi, __shfl_xor_sync(0xffffffffu, hi, o));
            lo = min_nan(lo, __shfl_xor_sync(0xffffffffu, lo, o));
        }
        const __half d    = q4_scale(hi, lo);
        const float  d32  = __half2float(d);
        const float  inv  = d32 == 0.0f ? 0.0f : __fdiv_rn(1.0f, d32);
        uint32_t     near = 0xFFFFFFFFu;
        uint32_t     c0 = q4_codes4(x, d32, inv, &near), c1 = q4_codes4(x + 4, d32, inv, &near);
        if (near < __float_as_uint(0x1p-18f) - 1u) {
            c0 = c1 = 0;
#pragma unroll 1
            for (int i = 0; i < 4; i++) {
                c0 = (c0 >> 8) | (q4_code(i == 0 ? x[0] : i == 1 ? x[1] : i == 2 ? x[2] : x[3], d32) << 24);
                c1 = (c1 >> 8) | (q4_code(i == 0 ? x[4] : i == 1 ? x[5] : i == 2 ? x[6] : x[7], d32) << 24);
            }
        }
        // lanes 0, 1 of a block hold its elements 0..15 (low halves of bytes 0..15), lanes 2, 3 the high halves: lane
        // 0 takes bytes 0..3, lane 2 bytes 4..7, lane 1 bytes 8..11, lane 3 bytes 12..15
        const bool     top  = sub & 2;
        const uint32_t far  = __shfl_xor_sync(0xffffffffu, top ? c0 : c1, 2);
        const uint32_t both = top ? far | (c1 << 4) : c0 | (far << 4);
        if (live && !bad) {
            const int64_t row = a.kv.row(pg, h, p);
            *reinterpret_cast<uint32_t *>(codes + row * (D / 2) + (sub >> 2) * 16 + (sub & 1) * 8 + (top ? 4 : 0)) = both;
            if ((sub & 3) == 0) {
                scales[row * (D / 32) + (sub >> 2)] = __half_as_ushort(d);
            }
        }
    };
    auto values = [&](int kind, int u, bool live, float * x) {
#pragma unroll
        for (int i = 0; i < 8; i++) {
            x[i] = live ? in[kind][u][i / VI].get(i % VI) : 0.0f;
        }
    };
    float x[8];
    if (a.q_norm) {
        weights(a.q_norm);
    }
    for (int r = r0; r < a.Nh; r += U * TURN) {
        if (r != r0) {
            load(0, r, a.Nh);
        }
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int h = r + u * TURN + rl;
            if (r + u * TURN < a.Nh) {
                values(0, u, h < a.Nh, x);
                norm_turn(x, a.q_norm);
                if (h < a.Nh) {
                    typename io<TQ>::t * q = reinterpret_cast<typename io<TQ>::t *>(a.q_out) + t * a.q_stride + h * D + d0;
#pragma unroll
                    for (int i = 0; i < 8 / VQ; i++) {
                        vec16<TQ> out;
#pragma unroll
                        for (int e = 0; e < VQ; e++) {
                            out.set(e, bad ? 0.0f : x[i * VQ + e]);
                        }
                        out.store(q + i * VQ);
                    }
                }
            }
        }
    }
    if (a.k_norm) {
        weights(a.k_norm);
    }
    for (int r = r0; r < a.kv.nkv; r += U * TURN) {
        if (r != r0) {
            load(1, r, a.kv.nkv);
            load(2, r, a.kv.nkv);
        }
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int h = r + u * TURN + rl;
            if (r + u * TURN < a.kv.nkv) {
                values(1, u, h < a.kv.nkv, x);
                norm_turn(x, a.k_norm);
                quantise(x, h < a.kv.nkv, h, a.kv.kc, a.kv.ks);
                values(2, u, h < a.kv.nkv, x);
                quantise(x, h < a.kv.nkv, h, a.kv.vc, a.kv.vs);
            }
        }
    }
}

// whether rows, norms and rotation fall on whole vectors of 8 elements
bool append_vector(const AppendArgs & a, int ti, int tq) {
    uintptr_t at = reinterpret_cast<uintptr_t>(a.qkv) | reinterpret_cast<uintptr_t>(a.q_out) | reinterpret_cast<uintptr_t>(a.q_norm) |
                   reinterpret_cast<uintptr_t>(a.k_norm) | reinterpret_cast<uintptr_t>(a.table);
    at |= (uintptr_t) (a.stride * type_size(ti)) | (uintptr_t) (a.Nh > 0 ? a.q_stride * type_size(tq) : 0);
    return at % 16 == 0 && (!a.table || a.R % (a.half ? 16 : 8) == 0);
}

// a thread 8 bytes of codes (16 elements, two runs of 8) of one row of k or v: items (token, kv head, k or v, half block)
template <int TO, int D>
__global__ void __launch_bounds__(256) kv_q4_read_kernel(const KvQ4 kv, const int32_t * __restrict__ seq,
                                                         const int32_t * __restrict__ pos, int64_t n_tok, void * k_out,
                                                         void * v_out, int64_t stride, bool vec, int * err) {
    constexpr int IPR  = D / 16;  // items of a row
    const uint32_t item = blockIdx.x * 256 + threadIdx.x;  // there are fewer than 2^31
    const uint32_t rows = item / IPR, per = 2 * (uint32_t) kv.nkv;
    const int      part = (int) (item % IPR), blk = part >> 1;
    const int64_t  t    = rows / per;
    if (t >= n_tok) {
        return;
    }
    const int  r = (int) (rows % per), h = r < kv.nkv ? r : r - kv.nkv;
    const bool is_v = r >= kv.nkv;
    void *        out  = is_v ? v_out : k_out;
    const int     s = __ldg(seq + t), p = __ldg(pos + t);
    if (s < 0 || !out) {
        return;
    }
    int bad = s >= kv.n_seq ? ACB_DEVERR_ID_RANGE : 0;
    if (p < 0 || (p >> kv.shift) >= kv.max_pages) {
        bad |= ACB_DEVERR_POS_RANGE;
    }
    const int pg = bad ? -1 : kv.page_of(s, p);
    if (!bad && pg < 0) {
        bad = ACB_DEVERR_PAGE_RANGE;
    }
    if (bad && part == 0 && err) {
        atomicOr(err, bad);
    }
    using E = typename io<TO>::t;
    E *   y = reinterpret_cast<E *>(out) + t * stride + (int64_t) h * D + blk * 32 + (part & 1) * 8;
    uint2 w = make_uint2(0x88888888u, 0x88888888u);
    float d = 0.0f;
    if (!bad) {
        const int64_t row = kv.row(pg, h, p);
        w                 = *reinterpret_cast<const uint2 *>((is_v ? kv.vc : kv.kc) + row * (D / 2) + part * 8);
        d                 = f16_bits_to_f(((is_v ? kv.vs : kv.ks) + row * (D / 32))[blk]);
    }
#pragma unroll
    for (int half = 0; half < 2; half++) {  // low halves: elements 0..15 of the block, high halves: 16..31
        float v[8];
#pragma unroll
        for (int e = 0; e < 8; e++) {
            const uint32_t c = ((e < 4 ? w.x : w.y) >> (8 * (e & 3) + 4 * half)) & 15u;
            v[e]             = __fmul_rn((float) (int) c - 8.0f, d);
        }
        if (vec) {
#pragma unroll
            for (int i = 0; i < 8 / vec16<TO>::N; i++) {
                vec16<TO> o;
#pragma unroll
                for (int e = 0; e < vec16<TO>::N; e++) {
                    o.set(e, v[i * vec16<TO>::N + e]);
                }
                o.store(y + half * 16 + i * vec16<TO>::N);
            }
        } else {
#pragma unroll
            for (int e = 0; e < 8; e++) {
                y[half * 16 + e] = io<TO>::from_f(v[e]);
            }
        }
    }
}

template <int TI, int TQ, int D> void (*append_vec(int rope))(const AppendArgs) {
    return rope == 0 ? kv_q4_append_vec_kernel<TI, TQ, D, 0> : rope == 1 ? kv_q4_append_vec_kernel<TI, TQ, D, 1>
                                                                         : kv_q4_append_vec_kernel<TI, TQ, D, 2>;
}

// rope < 0: the form through shared memory
template <int TI, int TQ> void (*append_kernel(int D, int rope))(const AppendArgs) {
    if (rope >= 0) {
        return D == 64 ? append_vec<TI, TQ, 64>(rope) : D == 128 ? append_vec<TI, TQ, 128>(rope) : append_vec<TI, TQ, 256>(rope);
    }
    return D == 64 ? kv_q4_append_kernel<TI, TQ, 64> : D == 128 ? kv_q4_append_kernel<TI, TQ, 128>
                                                                : kv_q4_append_kernel<TI, TQ, 256>;
}

template <int TI> void (*append_kernel(int tq, int D, int rope))(const AppendArgs) {
    return tq == ACB_TYPE_F32   ? append_kernel<TI, ACB_TYPE_F32>(D, rope)
           : tq == ACB_TYPE_F16 ? append_kernel<TI, ACB_TYPE_F16>(D, rope)
                                : append_kernel<TI, ACB_TYPE_BF16>(D, rope);
}

using ReadKernel = void (*)(const KvQ4, const int32_t *, const int32_t *, int64_t, void *, void *, int64_t, bool, int *);

template <int TO> ReadKernel read_kernel(int D) {
    return D == 64 ? kv_q4_read_kernel<TO, 64> : D == 128 ? kv_q4_read_kernel<TO, 128> : kv_q4_read_kernel<TO, 256>;
}

}  // namespace
}  // namespace acb

using namespace acb;

extern "C" acb_status acb_kv_q4_append(const acb_kv_q4 * kv, const void * qkv, int type, int64_t stride,
                                       int64_t n_tok, int n_heads, const float * q_norm, const float * k_norm,
                                       float eps, const float * rope_table, int max_pos, int rope_dim, int layout,
                                       const int32_t * seq, const int32_t * pos, void * q_out, int q_type,
                                       int64_t q_stride, int * err_flag, acb_stream_t stream) {
    AppendArgs       a  = {};
    const acb_status rc = kv_q4_check(kv, &a.kv);
    if (rc != ACB_OK) {
        return rc;
    }
    const int D = kv->head_dim;
    if (!qkv || !seq || !pos || n_tok < 0 || n_heads < 0 || (n_heads > 0 && !q_out)) {
        return ACB_ERR_INVALID_ARG;
    }
    const int64_t nh = (int64_t) n_heads + 2 * (int64_t) kv->n_kv_heads;
    if (stride < nh * D || (n_heads > 0 && q_stride < (int64_t) n_heads * D)) {
        return ACB_ERR_INVALID_ARG;
    }
    if (rope_table && (max_pos <= 0 || rope_dim < 2 || rope_dim > D || rope_dim % 2 != 0 ||
                       (layout != ACB_ROPE_HALF && layout != ACB_ROPE_INTERLEAVED))) {
        return ACB_ERR_INVALID_ARG;
    }
    if (!is_io_type(type) || (n_heads > 0 && !is_io_type(q_type)) || n_tok > std::min((int64_t) INT32_MAX, (int64_t) INT32_MAX * 8 / nh) ||
        nh * D > (int64_t) INT32_MAX) {  // the kernels count within a row in 32 bits
        return ACB_ERR_UNSUPPORTED;
    }
    if (n_heads > 0 && q_out == qkv && (q_type != type || (n_tok > 1 && q_stride != stride))) {
        return ACB_ERR_INVALID_ARG;  // one buffer in two layouts would be written before it is read
    }
    if (n_tok == 0) {
        return ACB_OK;
    }
    a.qkv      = qkv;
    a.stride   = stride;
    a.n_tok    = n_tok;
    a.Nh       = n_heads;
    a.q_norm   = q_norm;
    a.k_norm   = k_norm;
    a.eps      = eps;
    a.table    = rope_table;
    a.max_pos  = max_pos;
    a.R        = rope_dim;
    a.half     = layout == ACB_ROPE_HALF;
    a.seq      = seq;
    a.pos      = pos;
    a.q_out    = q_out;
    a.q_stride = q_stride;
    a.err      = err_flag;
    const int  tq   = n_heads > 0 ? q_type : type;
    const bool vec  = append_vector(a, type, tq);
    const int  rope = !vec ? -1 : !rope_table ? 0 : a.half ? 1 : 2;
    const auto kern = type == ACB_TYPE_F32   ? append_kernel<ACB_TYPE_F32>(tq, D, rope)
                      : type == ACB_TYPE_F16 ? append_kernel<ACB_TYPE_F16>(tq, D, rope)
                                             : append_kernel<ACB_TYPE_BF16>(tq, D, rope);
    if (vec) {
        // as many warps for a token as keep all tokens on the GPU at once: 8 tokens (16 + 8 + 8 heads of 128, bf16) take 4.2 us by
        // 4 warps and 11.2 by one, 1184 take 9.7 by 2 (10.8, 13.4 by 4, 1), and 8192 take 47 by one and 54 by 4
        int warps = kAppendWarps;
        while (warps > 1 && n_tok * warps > (int64_t) kAppendRoom * num_sms()) {
            warps /= 2;
        }
        kern<<<(unsigned) n_tok, 32 * warps, 0, (cudaStream_t) stream>>>(a);
    } else {
        kern<<<(unsigned) ((n_tok * nh + 7) / 8), 256, 0, (cudaStream_t) stream>>>(a);
    }
    return launch_status();
}

extern "C" acb_status acb_kv_q4_read(const acb_kv_q4 * kv, const int32_t * seq, const int32_t * pos, int64_t n_tok,
                                     void * k_out, void * v_out, int out_type, int64_t out_stride, int * err_flag,
                                     acb_stream_t stream) {
    KvQ4             d  = {};
    const acb_status rc = kv_q4_check(kv, &d);
    if (rc != ACB_OK) {
        return rc;
    }
    if (!seq || !pos || (!k_out && !v_out) || n_tok < 0 || out_stride < (int64_t) kv->n_kv_heads * kv->head_dim) {
        return ACB_ERR_INVALID_ARG;
    }
    if (!is_io_type(out_type) || n_tok > (int64_t) INT32_MAX * 8 / ((int64_t) kv->n_kv_heads * kv->head_dim)) {
        return ACB_ERR_UNSUPPORTED;
    }
    if (n_tok == 0) {
        return ACB_OK;
    }
    const ReadKernel kern = out_type == ACB_TYPE_F32   ? read_kernel<ACB_TYPE_F32>(kv->head_dim)
                            : out_type == ACB_TYPE_F16 ? read_kernel<ACB_TYPE_F16>(kv->head_dim)
                                                       : read_kernel<ACB_TYPE_BF16>(kv->head_dim);
    const bool vec = (reinterpret_cast<uintptr_t>(k_out) | reinterpret_cast<uintptr_t>(v_out)) % 16 == 0 &&
                     out_stride * type_size(out_type) % 16 == 0;
    const int64_t items = n_tok * 2 * kv->n_kv_heads * (kv->head_dim / 16);
    kern<<<(unsigned) ((items + 255) / 256), 256, 0, (cudaStream_t) stream>>>(d, seq, pos, n_tok, k_out, v_out, out_stride,
                                                                              vec, err_flag);
    return launch_status();
}
