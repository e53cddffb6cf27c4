// k_logits.cu -- rules on logits in front of the sampler (acb_logits_rules): repetition, frequency and presence
// penalties, a bias per token and a grammar mask, in one pass over the row.
//
// A block owns kLChunk columns of one row. It first counts, in shared memory, how often each of its columns occurs in the
// row's history (whole numbers, so the order of the atomics does not show) and notes the last bias entry of each; then every
// column is read, changed and written once. The row's bytes bound it: the history is short against it and comes
// from L2 after the first block.
#include "common.cuh"

namespace acb {
namespace {

constexpr int      kLChunk   = 4096;
constexpr int      kLThreads = 256;
constexpr uint32_t kInPrompt = 0x80000000u;  // column occurs in the prompt; the low bits count the answer

struct RulesArgs {
    const void *    x;
    int64_t         ld;
    void *          y;
    int64_t         ldo;
    int64_t         V;
    acb_logit_rules r;
    int *           err;
};

template <int TI, int TO> __global__ void __launch_bounds__(kLThreads) logits_rules_kernel(const RulesArgs a) {
    __shared__ uint32_t seen[kLChunk];
    __shared__ int32_t  bias[kLChunk];
    const int           row = blockIdx.y;
    const int64_t       c0  = (int64_t) blockIdx.x * kLChunk;
    const int           n   = (int) min((int64_t) kLChunk, a.V - c0);
    const bool          use_hist = a.r.hist != nullptr, use_bias = a.r.bias_ids != nullptr;
    for (int i = threadIdx.x; i < kLChunk; i += kLThreads) {
        seen[i] = 0;
        bias[i] = -1;
    }
    __syncthreads();
    int bad = 0;
    if (use_hist) {
        const int32_t * h   = a.r.hist + (int64_t) row * a.r.hist_stride;
        int64_t         len = a.r.hist_len ? (int64_t) __ldg(a.r.hist_len + row) : a.r.hist_stride;
        len                 = min(max(len, (int64_t) 0), a.r.hist_stride);
        const int64_t np    = a.r.prompt_len ? (int64_t) __ldg(a.r.prompt_len + row) : 0;
        for (int64_t i = threadIdx.x; i < len; i += kLThreads) {
            const int64_t v = __ldg(h + i);
            if (v >= a.V) {
                bad = 1;
            } else if (v >= c0 && v < c0 + n) {
                if (i < np) {
                    atomicOr(&seen[v - c0], kInPrompt);
                } else {
                    atomicAdd(&seen[v - c0], 1u);
                }
            }
        }
    }
    if (use_bias) {
        const int32_t * b = a.r.bias_ids + (int64_t) row * a.r.bias_stride;
        for (int i = threadIdx.x; i < a.r.n_bias; i += kLThreads) {
            const int64_t v = __ldg(b + i);
            if (v >= a.V) {
                bad = 1;
            } else if (v >= c0 && v < c0 + n) {
                atomicMax(&bias[v - c0], i);
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
    __syncthreads();
    const float rep  = a.r.rep ? __ldg(a.r.rep + row) : 1.0f;
    const float freq = a.r.freq ? __ldg(a.r.freq + row) : 0.0f;
    const float pres = a.r.pres ? __ldg(a.r.pres + row) : 0.0f;
    const typename io<TI>::t * x = reinterpret_cast<const typename io<TI>::t *>(a.x) + (int64_t) row * a.ld + c0;
    typename io<TO>::t *       y = reinterpret_cast<typename io<TO>::t *>(a.y) + (int64_t) row * a.ldo + c0;
    for (int i = threadIdx.x; i < n; i += kLThreads) {
        float          f = io<TI>::to_f(x[i]);
        const uint32_t c = seen[i];
        if (c) {
            if (a.r.rep) {
                f = f > 0.0f ? __fdiv_rn(f, rep) : __fmul_rn(f, rep);
            }
            const uint32_t k = c & ~kInPrompt;
            if (k) {
                f = __fsub_rn(__fsub_rn(f, __fmul_rn(freq, (float) k)), pres);
            }
        }
        if (bias[i] >= 0) {
            f = __fadd_rn(f, __ldg(a.r.bias_val + (int64_t) row * a.r.bias_stride + bias[i]));
        }
        const int64_t v = c0 + i;
        if (mask && !((__ldg(mask + (v >> 5)) >> (v & 31)) & 1u)) {
            f = -INFINITY;
        }
        y[i] = io<TO>::from_f(f);
    }
}

template <int TI> void (*rules_kernel(int to))(const RulesArgs) {
    return to == ACB_TYPE_F32   ? logits_rules_kernel<TI, ACB_TYPE_F32>
           : to == ACB_TYPE_F16 ? logits_rules_kernel<TI, ACB_TYPE_F16>
                                : logits_rules_kernel<TI, ACB_TYPE_BF16>;
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
    if (!is_io_type(type) || !is_io_type(out_type) || rows > 65535 || V > INT32_MAX || r.hist_stride > INT32_MAX) {
        return ACB_ERR_UNSUPPORTED;
    }
    if (rows == 0) {
        return ACB_OK;
    }
    const RulesArgs a    = { logits, ld, out, ld_out, V, r, err_flag };
    const auto      kern = type == ACB_TYPE_F32   ? rules_kernel<ACB_TYPE_F32>(out_type)
                           : type == ACB_TYPE_F16 ? rules_kernel<ACB_TYPE_F16>(out_type)
                                                  : rules_kernel<ACB_TYPE_BF16>(out_type);
    kern<<<dim3((unsigned) ((V + kLChunk - 1) / kLChunk), (unsigned) rows), kLThreads, 0, (cudaStream_t) stream>>>(a);
    return launch_status();
}
