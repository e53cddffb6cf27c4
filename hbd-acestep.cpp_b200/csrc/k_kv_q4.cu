// k_kv_q4.cu -- the writes of the paged 4-bit KV cache (acb_kv_q4_append: norm, rotation, quantisation and scatter in
// one pass over the fused qkv rows) and the rows read back as values (acb_kv_q4_read).
//
// A block of 32 values x is held as d (code - 8) with d = f16(bf16(-mx / 8)), mx the value of largest magnitude: mx itself
// gets code 0, its negative side reaches 15. Rounding d to bf16 (8 significant bits; 2^-9 of the block's largest value
// against the codes' own step of 2^-4) makes every product d (code - 8) an f16 number, because |code - 8| <= 8 has at most
// 3 significant bits: the attention's operands are then exact. The codes come from a correctly rounded division, so that a
// quotient that is exactly between two codes (16-bit inputs often are) goes the same way everywhere.
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

// one warp per (token, kv head, k or v)
template <int TO, int D>
__global__ void __launch_bounds__(256) kv_q4_read_kernel(const KvQ4 kv, const int32_t * __restrict__ seq,
                                                         const int32_t * __restrict__ pos, int64_t n_tok, void * k_out,
                                                         void * v_out, int64_t stride, int * err) {
    constexpr int E    = D / 32;
    const int     lane = threadIdx.x & 31;
    const int64_t item = (int64_t) blockIdx.x * 8 + (threadIdx.x >> 5);
    if (item >= n_tok * 2 * kv.nkv) {
        return;
    }
    const int64_t t = item / (2 * kv.nkv);
    const int     r = (int) (item - t * 2 * kv.nkv), h = r >> 1;
    const bool    is_v = r & 1;
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
    if (bad && lane == 0 && err) {
        atomicOr(err, bad);
    }
    typename io<TO>::t * y = reinterpret_cast<typename io<TO>::t *>(out) + t * stride + (int64_t) h * D;
    const int64_t        row = bad ? 0 : kv.row(pg, h, p);
#pragma unroll
    for (int e = 0; e < E; e++) {
        float v = 0.0f;
        if (!bad) {
            const uint32_t b = ((is_v ? kv.vc : kv.kc) + row * (D / 2))[e * 16 + (lane & 15)];
            const float    d = f16_bits_to_f(((is_v ? kv.vs : kv.ks) + row * E)[e]);
            v                = __fmul_rn((float) (int) (lane < 16 ? b & 15u : b >> 4) - 8.0f, d);
        }
        y[e * 32 + lane] = io<TO>::from_f(v);
    }
}

template <int TI, int TQ> void (*append_kernel(int D))(const AppendArgs) {
    return D == 64 ? kv_q4_append_kernel<TI, TQ, 64> : D == 128 ? kv_q4_append_kernel<TI, TQ, 128>
                                                                : kv_q4_append_kernel<TI, TQ, 256>;
}

template <int TI> void (*append_kernel(int tq, int D))(const AppendArgs) {
    return tq == ACB_TYPE_F32 ? append_kernel<TI, ACB_TYPE_F32>(D)
           : tq == ACB_TYPE_F16 ? append_kernel<TI, ACB_TYPE_F16>(D)
                                : append_kernel<TI, ACB_TYPE_BF16>(D);
}

using ReadKernel = void (*)(const KvQ4, const int32_t *, const int32_t *, int64_t, void *, void *, int64_t, int *);

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
    if (!is_io_type(type) || (n_heads > 0 && !is_io_type(q_type)) || n_tok > (int64_t) INT32_MAX * 8 / nh) {
        return ACB_ERR_UNSUPPORTED;
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
    const auto kern = type == ACB_TYPE_F32   ? append_kernel<ACB_TYPE_F32>(tq, D)
                      : type == ACB_TYPE_F16 ? append_kernel<ACB_TYPE_F16>(tq, D)
                                             : append_kernel<ACB_TYPE_BF16>(tq, D);
    kern<<<(unsigned) ((n_tok * nh + 7) / 8), 256, 0, (cudaStream_t) stream>>>(a);
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
    if (!is_io_type(out_type) || n_tok > (int64_t) INT32_MAX * 4 / kv->n_kv_heads) {
        return ACB_ERR_UNSUPPORTED;
    }
    if (n_tok == 0) {
        return ACB_OK;
    }
    const ReadKernel kern = out_type == ACB_TYPE_F32   ? read_kernel<ACB_TYPE_F32>(kv->head_dim)
                            : out_type == ACB_TYPE_F16 ? read_kernel<ACB_TYPE_F16>(kv->head_dim)
                                                       : read_kernel<ACB_TYPE_BF16>(kv->head_dim);
    kern<<<(unsigned) ((n_tok * 2 * kv->n_kv_heads + 7) / 8), 256, 0, (cudaStream_t) stream>>>(
        d, seq, pos, n_tok, k_out, v_out, out_stride, err_flag);
    return launch_status();
}
