// k_attn_q4.cu -- causal attention over the paged 4-bit KV cache (acb_attn_kv_q4).
//
// One pass over the keys with the running maximum m and sum l of the softmax: for a new score s, m' = max(m, s),
// l' = l e^(m - m') + e^(s - m'), o' = o e^(m - m') + e^(s - m') v; the output is o / l.
#include "kv_q4.cuh"

namespace acb {
namespace {

struct AttnQ4Args {
    const void *    q;
    int64_t         q_stride, n_tok;
    int             Nh;
    const int32_t * q_start;
    const int32_t * kv_len;
    int             max_q, max_kv, window;
    float           scale_log2;
    void *          o;
    int64_t         o_stride;
    int *           err;
    KvQ4            kv;
};

// rows and keys of sequence s as the device arrays give them; false (and the error recorded by one thread of one block) when
// they are outside the call's bounds
__device__ __forceinline__ bool seq_bounds(const AttnQ4Args & a, int s, int64_t * row0, int * n, int * len) {
    const int64_t q0 = a.q_start ? __ldg(a.q_start + s) : s;
    const int64_t q1 = a.q_start ? __ldg(a.q_start + s + 1) : s + 1;
    *len             = __ldg(a.kv_len + s);
    *row0            = q0;
    *n               = (int) min((int64_t) a.max_q, max((int64_t) 0, q1 - q0));
    return q0 >= 0 && q1 >= q0 && q1 <= a.n_tok && q1 - q0 <= a.max_q && *len >= 0 && *len <= a.max_kv;
}

// one block per (row of a sequence, head), four warps, each taking every fourth key; a lane holds D/32 elements
template <int T, int D> __global__ void __launch_bounds__(128) attn_q4_kernel(const AttnQ4Args a) {
    constexpr int E = D / 32;
    const int     lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int     i = blockIdx.x, h = blockIdx.y, s = blockIdx.z;
    int64_t       row0;
    int           n, len;
    const bool    ok = seq_bounds(a, s, &row0, &n, &len);
    if (!ok && a.err && threadIdx.x == 0) {
        atomicOr(a.err, ACB_DEVERR_LEN_RANGE);
    }
    const int64_t t = row0 + i;
    if (i >= n || t < 0 || t >= a.n_tok) {
        return;
    }
    const int p  = ok ? len - n + i : -1;
    const int j0 = a.window > 0 ? max(0, p - a.window + 1) : 0;
    const int hk = h / (a.Nh / a.kv.nkv);
    using T1     = typename io<T>::t;
    const T1 * q = reinterpret_cast<const T1 *>(a.q) + t * a.q_stride + (int64_t) h * D;
    float      qv[E], o[E], m = -INFINITY, l = 0.0f;
    const int  b = lane & 15;
#pragma unroll
    for (int e = 0; e < E; e++) {
        qv[e] = io<T>::to_f(q[e * 32 + lane]) * a.scale_log2;
        o[e]  = 0.0f;
    }
    for (int j = j0 + warp; j <= p; j += 4) {
        const int pg = a.kv.page_of(s, j);
        if (pg < 0) {
            if (lane == 0 && a.err) {
                atomicOr(a.err, ACB_DEVERR_PAGE_RANGE);
            }
            continue;
        }
        const int64_t row = a.kv.row(pg, hk, j);
        float         sc = 0.0f, v[E];
#pragma unroll
        for (int e = 0; e < E; e++) {
            const uint32_t ck = a.kv.kc[row * (D / 2) + e * 16 + b], cv = a.kv.vc[row * (D / 2) + e * 16 + b];
            const float    kx = (float) (int) (lane < 16 ? ck & 15u : ck >> 4) - 8.0f;
            const float    vx = (float) (int) (lane < 16 ? cv & 15u : cv >> 4) - 8.0f;
            sc += qv[e] * kx * f16_bits_to_f(a.kv.ks[row * E + e]);
            v[e] = vx * f16_bits_to_f(a.kv.vs[row * E + e]);
        }
        sc            = warp_sum(sc);
        const float m1 = fmaxf(m, sc);
        const float al = m1 == -INFINITY ? 1.0f : exp2f(m - m1), pr = m1 == -INFINITY ? 0.0f : exp2f(sc - m1);
        m             = m1;
        l             = l * al + pr;
#pragma unroll
        for (int e = 0; e < E; e++) {
            o[e] = o[e] * al + pr * v[e];
        }
    }
    __shared__ float so[4][D], sm[4], sl[4];
#pragma unroll
    for (int e = 0; e < E; e++) {
        so[warp][e * 32 + lane] = o[e];
    }
    if (lane == 0) {
        sm[warp] = m;
        sl[warp] = l;
    }
    __syncthreads();
    const float M = fmaxf(fmaxf(sm[0], sm[1]), fmaxf(sm[2], sm[3]));
    T1 *        y = reinterpret_cast<T1 *>(a.o) + t * a.o_stride + (int64_t) h * D;
    for (int d = threadIdx.x; d < D; d += 128) {
        float L = 0.0f, r = 0.0f;
        for (int w = 0; w < 4; w++) {
            const float f = M == -INFINITY ? 0.0f : exp2f(sm[w] - M);
            L += f * sl[w];
            r += f * so[w][d];
        }
        y[d] = io<T>::from_f(L > 0.0f ? r / L : (L == L ? 0.0f : L));
    }
}

template <int T> void (*attn_kernel(int D))(const AttnQ4Args) {
    return D == 64 ? attn_q4_kernel<T, 64> : D == 128 ? attn_q4_kernel<T, 128> : attn_q4_kernel<T, 256>;
}

}  // namespace
}  // namespace acb

using namespace acb;

extern "C" size_t acb_attn_kv_q4_work_bytes(const acb_kv_q4 * kv, int64_t n_tok, int n_heads, int max_q_len,
                                            int max_kv_len) {
    return 0;
}

extern "C" acb_status acb_attn_kv_q4(const acb_kv_q4 * kv, const void * q, int type, int64_t q_stride, int64_t n_tok,
                                     int n_heads, const int32_t * q_start, const int32_t * kv_len, int max_q_len,
                                     int max_kv_len, int window, float scale, void * o, int64_t o_stride, void * work,
                                     size_t work_bytes, int * err_flag, acb_stream_t stream) {
    AttnQ4Args       a  = {};
    const acb_status rc = kv_q4_check(kv, &a.kv);
    if (rc != ACB_OK) {
        return rc;
    }
    if (!q || !o || !kv_len || n_tok < 0 || n_heads <= 0 || n_heads % kv->n_kv_heads != 0 || max_q_len <= 0 ||
        max_kv_len < 0 || window < 0 || !(scale == scale) || q_stride < (int64_t) n_heads * kv->head_dim ||
        o_stride < (int64_t) n_heads * kv->head_dim || (!q_start && (n_tok != kv->n_seq || max_q_len != 1))) {
        return ACB_ERR_INVALID_ARG;
    }
    if (max_kv_len > (int64_t) kv->max_pages * kv->page_size) {
        return ACB_ERR_OUT_OF_RANGE;
    }
    if (!is_io_type(type) || n_heads > 65535 || kv->n_seq > 65535) {
        return ACB_ERR_UNSUPPORTED;
    }
    if (n_tok == 0) {
        return ACB_OK;
    }
    a.q          = q;
    a.q_stride   = q_stride;
    a.n_tok      = n_tok;
    a.Nh         = n_heads;
    a.q_start    = q_start;
    a.kv_len     = kv_len;
    a.max_q      = max_q_len;
    a.max_kv     = max_kv_len;
    a.window     = window;
    a.scale_log2 = scale * 1.4426950408889634f;
    a.o          = o;
    a.o_stride   = o_stride;
    a.err        = err_flag;
    const auto kern = type == ACB_TYPE_F32   ? attn_kernel<ACB_TYPE_F32>(kv->head_dim)
                      : type == ACB_TYPE_F16 ? attn_kernel<ACB_TYPE_F16>(kv->head_dim)
                                             : attn_kernel<ACB_TYPE_BF16>(kv->head_dim);
    kern<<<dim3((unsigned) max_q_len, (unsigned) n_heads, (unsigned) kv->n_seq), 128, 0, (cudaStream_t) stream>>>(a);
    return launch_status();
}
