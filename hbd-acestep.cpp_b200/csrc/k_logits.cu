// k_logits.cu -- rules on logits in front of the sampler (acb_logits_rules): repetition, frequency and presence
// penalties, a bias per token and a grammar mask, in one pass over the row.
//
// A block owns a chunk of columns of one row, each thread kLCols of them, whose logits are under way before anything else is
// done. A 32-bit word per column in shared memory then takes the last bias entry of the column (its number + 1 above kBiasBit, by
// a maximum), whether the prompt holds it, and how often the answer does (whole numbers, so the order of the atomics does not
// show). The row's bytes bound it; the history is short against them, but every block of the row reads it, so the chunks are
// large, except where a call of few rows would leave SMs idle.
#include "common.cuh"

namespace acb {
namespace {

constexpr int      kLCols     = 16;
constexpr int      kBiasBit   = 21;
constexpr uint32_t kInPrompt  = 1u << 20;
constexpr uint32_t kCountMask = kInPrompt - 1;  // histories and bias lists are limited to what the fields hold

struct RulesArgs {
    const void *    x;
    int64_t         ld;
    void *          y;
    int64_t         ldo;
    int64_t         V;
    acb_logit_rules r;
    int *           err;
};

// VEC: rows are 16-byte aligned on both sides and V is a multiple of 8, so a thread's columns are whole vectors of 8
template <int TI, int TO, int THREADS, bool VEC>
__global__ void __launch_bounds__(THREADS) logits_rules_kernel(const RulesArgs a) {
    constexpr int       C = THREADS * kLCols, G = kLCols / 8;
    using EI              = typename io<TI>::t;
    using EO              = typename io<TO>::t;
    __shared__ uint32_t tab[C];
    const int           row = blockIdx.y, tid = threadIdx.x;
    const int64_t       c0  = (int64_t) blockIdx.x * C;
    const int           n   = (int) min((int64_t) C, a.V - c0);
    const EI *          x   = reinterpret_cast<const EI *>(a.x) + (int64_t) row * a.ld + c0;
    EO *                y   = reinterpret_cast<EO *>(a.y) + (int64_t) row * a.ldo + c0;
    // column of element e of group g: vectors of 8 in turn over the threads, or single columns
    auto     col = [&](int g, int e) { return VEC ? (g * THREADS + tid) * 8 + e : (g * 8 + e) * THREADS + tid; };
    vec16<TI> in[G][8 / vec16<TI>::N];
    float     f[VEC ? 1 : G][8];
#pragma unroll
    for (int g = 0; g < G; g++) {
        if constexpr (VEC) {
            if (col(g, 0) < n) {
#pragma unroll
                for (int v = 0; v < 8 / vec16<TI>::N; v++) {
                    in[g][v].load(x + col(g, v * vec16<TI>::N));
                }
            }
        } else {
#pragma unroll
            for (int e = 0; e < 8; e++) {
                f[g][e] = col(g, e) < n ? io<TI>::to_f(x[col(g, e)]) : 0.0f;
            }
        }
    }
    const bool use = a.r.hist != nullptr || a.r.bias_ids != nullptr;
    int        bad = 0;
    if (use) {
        for (int i = tid; i < C / 4; i += THREADS) {
            reinterpret_cast<uint4 *>(tab)[i] = make_uint4(0, 0, 0, 0);
        }
        __syncthreads();
    }
    if (a.r.bias_ids) {
        const int32_t * b = a.r.bias_ids + (int64_t) row * a.r.bias_stride;
        for (int i = tid; i < a.r.n_bias; i += THREADS) {
            const int64_t v = __ldg(b + i);
            if (v >= a.V) {
                bad = 1;
            } else if (v >= c0 && v < c0 + n) {
                atomicMax(&tab[v - c0], (uint32_t) (i + 1) << kBiasBit);
            }
        }
        __syncthreads();
    }
    if (a.r.hist) {
        const int32_t * h   = a.r.hist + (int64_t) row * a.r.hist_stride;
        int             len = a.r.hist_len ? __ldg(a.r.hist_len + row) : (int) a.r.hist_stride;
        len                 = min(max(len, 0), (int) a.r.hist_stride);
        const int np        = a.r.prompt_len ? __ldg(a.r.prompt_len + row) : 0;
        constexpr int U     = 8;  // tokens in flight per thread
        for (int i0 = 0; i0 < len; i0 += THREADS * U) {
            int v[U];
#pragma unroll
            for (int u = 0; u < U; u++) {
                const int i = i0 + u * THREADS + tid;
                v[u]        = i < len ? __ldg(h + i) : -1;
            }
#pragma unroll
            for (int u = 0; u < U; u++) {
                bad |= v[u] >= a.V;
                const int64_t k = (int64_t) v[u] - c0;
                if (k >= 0 && k < n) {
                    if (i0 + u * THREADS + tid < np) {
                        atomicOr(&tab[k], kInPrompt);
                    } else {
                        atomicAdd(&tab[k], 1u);
                    }
                }
            }
        }
    }
    const uint32_t * mask = nullptr;
    if (a.r.mask) {
        const int mr = a.r.mask_row ? __ldg(a.r.mask_row + row) : row;
        if (mr >= a.r.n_masks) {
            bad = 1;
        } else if (mr >= 0) {
            mask = a.r.mask + (int64_t) mr * a.r.mask_stride;
        }
    }
    if (bad && a.err) {
        atomicOr(a.err, ACB_DEVERR_ID_RANGE);
    }
    const float rep  = a.r.rep ? __ldg(a.r.rep + row) : 1.0f;
    const float freq = a.r.freq ? __ldg(a.r.freq + row) : 0.0f;
    const float pres = a.r.pres ? __ldg(a.r.pres + row) : 0.0f;
    if (use) {
        __syncthreads();
    }
    auto change = [&](float v, uint32_t w) {
        if (w) {
            if (w & (kInPrompt | kCountMask)) {
                if (a.r.rep) {
                    v = v > 0.0f ? __fdiv_rn(v, rep) : __fmul_rn(v, rep);
                }
                const uint32_t k = w & kCountMask;
                if (k) {
                    v = __fsub_rn(__fsub_rn(v, __fmul_rn(freq, (float) k)), pres);
                }
            }
            if (w >> kBiasBit) {
                v = __fadd_rn(v, __ldg(a.r.bias_val + (int64_t) row * a.r.bias_stride + (w >> kBiasBit) - 1));
            }
        }
        return v;
    };
#pragma unroll
    for (int g = 0; g < G; g++) {
        if constexpr (VEC) {
            const int c = col(g, 0);
            if (c >= n) {
                continue;
            }
            float v[8];
#pragma unroll
            for (int e = 0; e < 8; e++) {
                v[e] = in[g][e / vec16<TI>::N].get(e % vec16<TI>::N);
            }
            if (use) {
                const uint4 w0 = *reinterpret_cast<const uint4 *>(tab + c), w1 = *reinterpret_cast<const uint4 *>(tab + c + 4);
                if (w0.x | w0.y | w0.z | w0.w | w1.x | w1.y | w1.z | w1.w) {
                    const uint32_t w[8] = { w0.x, w0.y, w0.z, w0.w, w1.x, w1.y, w1.z, w1.w };
#pragma unroll
                    for (int e = 0; e < 8; e++) {
                        v[e] = change(v[e], w[e]);
                    }
                }
            }
            if (mask) {
                const uint32_t m = __ldg(mask + ((c0 + c) >> 5)) >> ((c0 + c) & 31);
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    v[e] = (m >> e) & 1u ? v[e] : -INFINITY;
                }
            }
            vec16<TO> out;
#pragma unroll
            for (int q = 0; q < 8 / vec16<TO>::N; q++) {
#pragma unroll
                for (int e = 0; e < vec16<TO>::N; e++) {
                    out.set(e, v[q * vec16<TO>::N + e]);
                }
                out.store(y + c + q * vec16<TO>::N);
            }
        } else {
#pragma unroll
            for (int e = 0; e < 8; e++) {
                const int c = col(g, e);
                if (c < n) {
                    float v = use ? change(f[g][e], tab[c]) : f[g][e];
                    if (mask && !((__ldg(mask + ((c0 + c) >> 5)) >> ((c0 + c) & 31)) & 1u)) {
                        v = -INFINITY;
                    }
                    y[c] = io<TO>::from_f(v);
                }
            }
        }
    }
}

template <int TI, int TO> void rules_launch(const RulesArgs & a, int rows, cudaStream_t st) {
    const bool vec = (reinterpret_cast<uintptr_t>(a.x) | reinterpret_cast<uintptr_t>(a.y)) % 16 == 0 &&
                     (a.ld * type_size(TI) | a.ldo * type_size(TO)) % 16 == 0 && a.V % 8 == 0;
    // 8192 columns a block; 2048 where that leaves SMs without a block
    const bool    few = (a.V + 8191) / 8192 * rows < num_sms();
    const int     c   = few ? 128 * kLCols : 512 * kLCols;
    const dim3    grid((unsigned) ((a.V + c - 1) / c), (unsigned) rows);
    if (few) {
        (vec ? logits_rules_kernel<TI, TO, 128, true> : logits_rules_kernel<TI, TO, 128, false>)<<<grid, 128, 0, st>>>(a);
    } else {
        (vec ? logits_rules_kernel<TI, TO, 512, true> : logits_rules_kernel<TI, TO, 512, false>)<<<grid, 512, 0, st>>>(a);
    }
}

template <int TI> void rules_launch(const RulesArgs & a, int to, int rows, cudaStream_t st) {
    if (to == ACB_TYPE_F32) {
        rules_launch<TI, ACB_TYPE_F32>(a, rows, st);
    } else if (to == ACB_TYPE_F16) {
        rules_launch<TI, ACB_TYPE_F16>(a, rows, st);
    } else {
        rules_launch<TI, ACB_TYPE_BF16>(a, rows, st);
    }
}

}  // namespace
}  // namespace acb

using namespace acb;

extern "C" acb_status acb_logits_rules(const void * logits, int type, int64_t ld, void * out, int out_type,
                                       int64_t ld_out, int rows, int64_t V, const acb_logit_rules * rules,
                                       int * err_flag, acb_stream_t stream) {
    if (!logits || !out || !rules || rows < 0 || V <= 0 || ld < V || ld_out < V) {
        return ACB_ERR_INVALID_ARG;
    }
    const acb_logit_rules & r = *rules;
    if ((r.hist && r.hist_stride < 0) || (!r.hist && (r.rep || r.freq || r.pres)) ||
        ((r.bias_ids != nullptr) != (r.bias_val != nullptr)) ||
        (r.bias_ids && (r.n_bias < 0 || (r.bias_stride != 0 && r.bias_stride < r.n_bias))) ||
        (r.mask && (r.n_masks <= 0 || r.mask_stride < (V + 31) / 32)) || (r.mask_row && !r.mask)) {
        return ACB_ERR_INVALID_ARG;
    }
    if (logits == out && (type != out_type || ld != ld_out)) {
        return ACB_ERR_INVALID_ARG;  // one buffer in two layouts would be written before it is read
    }
    if (!is_io_type(type) || !is_io_type(out_type) || rows > 65535 || V > (1 << 30) ||
        (r.hist && r.hist_stride > (int64_t) kCountMask) || (r.bias_ids && r.n_bias >= 1 << (32 - kBiasBit))) {
        return ACB_ERR_UNSUPPORTED;
    }
    if (rows == 0) {
        return ACB_OK;
    }
    const RulesArgs a  = { logits, ld, out, ld_out, V, r, err_flag };
    cudaStream_t    st = (cudaStream_t) stream;
    if (type == ACB_TYPE_F32) {
        rules_launch<ACB_TYPE_F32>(a, out_type, rows, st);
    } else if (type == ACB_TYPE_F16) {
        rules_launch<ACB_TYPE_F16>(a, out_type, rows, st);
    } else {
        rules_launch<ACB_TYPE_BF16>(a, out_type, rows, st);
    }
    return launch_status();
}
