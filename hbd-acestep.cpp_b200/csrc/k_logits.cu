// k_logits.cu -- rules on logits in front of the sampler (acb_logits_rules): repetition, frequency and presence
// penalties, a bias per token and a grammar mask, in one pass over the row.
//
// A block owns a slice of one row. It notes in shared memory what the history and the bias list say of its columns, streams the
// slice through (as it is, or -inf where the mask is closed), and then changes the few columns that were noted, a thread each.
// The row's bytes bound it. f32 rows are written 32 bytes a thread at once: in two stores of 16, each half of a sector, the plain
// stream of 128 rows of 151936 (bf16 to f32) takes 26 us, in one 18.7 (6.2 TB/s). The history is read once by every block of
// its row, so there are only as many slices as fill the GPU: cut into 19 slices a row, the histories of 128 rows were over
// half of the work (49-62 us in four forms). With all rules and histories of up to 4100 tokens the slices take 28.4 us: four
// warps note beside the stream, and the noted columns follow it. All warps streaming once they have noted gave nothing (30), nor
// did a second kernel that notes while the first streams (40).
//
// A column's word holds the last bias entry of the column (its number + 1 above kBiasBit, by a maximum), whether the prompt
// has it, and how often the answer does: whole numbers, so the order of the atomics does not show. The words are found by
// hashing where the history is short enough for it (the slice's distinct tokens are then at most 3/4 of the slots);
// otherwise the slice is gone through in parts of kWords columns with a word for each column.
#include "common.cuh"

namespace acb {
namespace {

constexpr int      kLThreads  = 512;
constexpr int      kWords     = 16384;        // 64 KB
constexpr int      kSlotsMost = kWords / 2;   // of the hash: a column and its word each
constexpr int      kHashMost  = kSlotsMost / 4 * 3;
constexpr int      kBiasBit   = 21;
constexpr uint32_t kInPrompt  = 1u << 20;
constexpr uint32_t kCountMask = kInPrompt - 1;  // histories and bias lists are limited to what the fields hold
constexpr uint32_t kNoColumn  = 0xFFFFFFFFu;

// 8 elements of a row, whole sectors at once where they are 32 bytes on their boundary
template <int T> __device__ __forceinline__ void store8(typename io<T>::t * y, const float * v, bool wide) {
    if constexpr (T == ACB_TYPE_F32) {
        if (wide) {
            asm volatile("st.global.v8.f32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(y), "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]),
                         "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7])
                         : "memory");
            return;
        }
    }
#pragma unroll
    for (int q = 0; q < 8 / vec16<T>::N; q++) {
        vec16<T> out;
#pragma unroll
        for (int e = 0; e < vec16<T>::N; e++) {
            out.set(e, v[q * vec16<T>::N + e]);
        }
        out.store(y + q * vec16<T>::N);
    }
}

struct RulesArgs {
    const void *    x;
    int64_t         ld;
    void *          y;
    int64_t         ldo;
    int64_t         V;
    acb_logit_rules r;
    int *           err;
    int             slice;   // columns of a block, a multiple of 256
    int             noters;  // threads that go through the history and the bias list
    int             slots, shift;  // of the hash: 2^(32 - shift)
};

// VEC: rows are 16-byte aligned on both sides and V is a multiple of 8
template <int TI, int TO, bool VEC, bool HASH>
__global__ void __launch_bounds__(kLThreads, 2) logits_rules_kernel(const RulesArgs a) {
    using EI = typename io<TI>::t;
    using EO = typename io<TO>::t;
    extern __shared__ uint32_t words[];
    __shared__ uint16_t        taken[HASH ? kHashMost : 1];  // slots in use, so that the change runs with full warps
    __shared__ int             n_taken;
    const int     row = blockIdx.y, tid = threadIdx.x;
    const int64_t c0  = (int64_t) blockIdx.x * a.slice;
    const int     n   = (int) min((int64_t) a.slice, a.V - c0);
    const EI *    x   = reinterpret_cast<const EI *>(a.x) + (int64_t) row * a.ld + c0;
    EO *          y   = reinterpret_cast<EO *>(a.y) + (int64_t) row * a.ldo + c0;
    const int32_t * hist = a.r.hist ? a.r.hist + (int64_t) row * a.r.hist_stride : nullptr;
    const int32_t * bids = a.r.bias_ids ? a.r.bias_ids + (int64_t) row * a.r.bias_stride : nullptr;
    const int       n_bias = bids ? a.r.n_bias : 0;
    int             len    = hist ? (int) a.r.hist_stride : 0;
    if (hist && a.r.hist_len) {
        len = min(max(__ldg(a.r.hist_len + row), 0), len);
    }
    const int        np   = a.r.prompt_len ? __ldg(a.r.prompt_len + row) : 0;
    const int        mr   = !a.r.mask ? -1 : a.r.mask_row ? __ldg(a.r.mask_row + row) : row;
    const uint32_t * mask = mr >= 0 && mr < a.r.n_masks ? a.r.mask + (int64_t) mr * a.r.mask_stride + (c0 >> 5) : nullptr;
    bool             bad  = a.r.mask && mr >= a.r.n_masks;
    const float      rep  = a.r.rep ? __ldg(a.r.rep + row) : 1.0f;
    const float      freq = a.r.freq ? __ldg(a.r.freq + row) : 0.0f;
    const float      pres = a.r.pres ? __ldg(a.r.pres + row) : 0.0f;

    // the word of column k of the slice while columns [k0, k1) are looked at; nullptr outside
    auto word_of = [&](int64_t v, int k0, int k1) -> uint32_t * {
        bad |= v >= a.V;
        const int64_t k = v - c0;
        if (k < k0 || k >= k1) {
            return nullptr;
        }
        if constexpr (HASH) {
            uint32_t s = ((uint32_t) k * 2654435761u) >> a.shift;
            for (;;) {  // ends: there are fewer columns than slots
                const uint32_t old = atomicCAS(&words[s], kNoColumn, (uint32_t) k);
                if (old == kNoColumn) {
                    taken[atomicAdd(&n_taken, 1)] = (uint16_t) s;
                }
                if (old == kNoColumn || old == (uint32_t) k) {
                    return &words[a.slots + s];
                }
                s = (s + 1) & (a.slots - 1);
            }
        }
        return &words[k - k0];
    };
    // Of U tokens at once (none where v < 0), by whole warps: what each would wait for, all wait for together, and the slots
    // that are new cost a warp one addition. One after the other, four warps took 20 us for 4100 tokens.
    constexpr int U = 8;
    auto words_of = [&](const int * v, uint32_t ** w) {
        uint32_t k[U], s[U], old[U], fresh[U];
        int      n_fresh = 0, to = 0;
#pragma unroll
        for (int u = 0; u < U; u++) {
            bad |= v[u] >= a.V;
            const int64_t at = v[u] - c0;
            k[u]             = v[u] >= 0 && at >= 0 && at < n ? (uint32_t) at : kNoColumn;
            s[u]             = (k[u] * 2654435761u) >> a.shift;
            old[u]           = k[u] == kNoColumn ? k[u] : atomicCAS(&words[s[u]], kNoColumn, k[u]);
        }
#pragma unroll
        for (int u = 0; u < U; u++) {
            while (k[u] != kNoColumn && old[u] != kNoColumn && old[u] != k[u]) {
                s[u]   = (s[u] + 1) & (a.slots - 1);
                old[u] = atomicCAS(&words[s[u]], kNoColumn, k[u]);
            }
        }
#pragma unroll
        for (int u = 0; u < U; u++) {
            fresh[u] = __ballot_sync(0xffffffffu, k[u] != kNoColumn && old[u] == kNoColumn);
            n_fresh += __popc(fresh[u]);
        }
        if ((tid & 31) == 0) {
            to = atomicAdd(&n_taken, n_fresh);
        }
        to = __shfl_sync(0xffffffffu, to, 0);
#pragma unroll
        for (int u = 0; u < U; u++) {
            if ((fresh[u] >> (tid & 31)) & 1u) {
                taken[to + __popc(fresh[u] & ((1u << (tid & 31)) - 1))] = (uint16_t) s[u];
            }
            to += __popc(fresh[u]);
            w[u] = k[u] == kNoColumn ? nullptr : &words[a.slots + s[u]];
        }
    };
    const int  nt   = a.noters;
    auto       sync = [&] { asm volatile("bar.sync 1, %0;" ::"r"(nt) : "memory"); };
    auto       note = [&](int k0, int k1) {  // called by the first nt threads
        const int m = HASH ? 2 * a.slots : kWords;
        if (tid == 0) {
            n_taken = 0;
        }
        for (int i = 4 * tid; i < m; i += 4 * nt) {
            const uint32_t z                       = HASH && i < a.slots ? kNoColumn : 0u;
            *reinterpret_cast<uint4 *>(words + i) = make_uint4(z, z, z, z);
        }
        sync();
        if (HASH && nt < kLThreads) {
            int        v[U];
            uint32_t * w[U];
            auto       take = [&](const int32_t * list, int i, int m) {
#pragma unroll
                for (int u = 0; u < U; u++) {
                    v[u] = i + u * nt < m ? __ldg(list + i + u * nt) : -1;
                }
            };
            for (int i0 = 0; i0 < n_bias; i0 += U * nt) {
                take(bids, i0 + tid, n_bias);
                words_of(v, w);
#pragma unroll
                for (int u = 0; u < U; u++) {
                    if (w[u]) {
                        atomicMax(w[u], (uint32_t) (i0 + tid + u * nt + 1) << kBiasBit);
                    }
                }
            }
            if (n_bias > 0) {
                sync();
            }
            for (int i0 = 0; i0 < len; i0 += U * nt) {
                take(hist, i0 + tid, len);
                words_of(v, w);
#pragma unroll
                for (int u = 0; u < U; u++) {
                    if (w[u]) {
                        if (i0 + tid + u * nt < np) {
                            atomicOr(w[u], kInPrompt);
                        } else {
                            atomicAdd(w[u], 1u);
                        }
                    }
                }
            }
            return;
        }
        for (int i = tid; i < n_bias; i += nt) {
            if (uint32_t * w = word_of(__ldg(bids + i), k0, k1)) {
                atomicMax(w, (uint32_t) (i + 1) << kBiasBit);
            }
        }
        if (n_bias > 0) {
            sync();  // a maximum of whole words: before anything is counted in them
        }
        for (int i0 = tid; i0 < len; i0 += U * nt) {
            int v[U];
#pragma unroll
            for (int u = 0; u < U; u++) {
                v[u] = i0 + u * nt < len ? __ldg(hist + i0 + u * nt) : -1;
            }
#pragma unroll
            for (int u = 0; u < U; u++) {
                if (uint32_t * w = word_of(v[u], k0, k1)) {
                    if (i0 + u * nt < np) {
                        atomicOr(w, kInPrompt);
                    } else {
                        atomicAdd(w, 1u);
                    }
                }
            }
        }
    };
    // (in place, an open column still holds its logit when this comes: it was written as it was)
    auto changed = [&](float v, uint32_t w) {
        if (w & (kInPrompt | kCountMask)) {
            if (a.r.rep) {
                v = v > 0.0f ? __fdiv_rn(v, rep) : __fmul_rn(v, rep);
            }
            const uint32_t times = w & kCountMask;
            if (times) {
                v = __fsub_rn(__fsub_rn(v, __fmul_rn(freq, (float) times)), pres);
            }
        }
        if (w >> kBiasBit) {
            v = __fadd_rn(v, __ldg(a.r.bias_val + (int64_t) row * a.r.bias_stride + (w >> kBiasBit) - 1));
        }
        return v;
    };
    // m words found by at(i, &column), i of this thread's share: logits and masks of several at once, since each comes from far
    auto change = [&](int m, auto at) {
        for (int i0 = tid; i0 < m; i0 += U * kLThreads) {
            int      k[U];
            uint32_t w[U], open[U];
            float    v[U];
#pragma unroll
            for (int u = 0; u < U; u++) {
                k[u] = 0;
                w[u] = i0 + u * kLThreads < m ? at(i0 + u * kLThreads, &k[u]) : 0u;
                if (w[u]) {
                    v[u]    = io<TI>::to_f(x[k[u]]);
                    open[u] = mask ? __ldg(mask + (k[u] >> 5)) >> (k[u] & 31) : 1u;
                }
            }
#pragma unroll
            for (int u = 0; u < U; u++) {
                if (w[u] && (open[u] & 1u)) {
                    y[k[u]] = io<TO>::from_f(changed(v[u], w[u]));
                }
            }
        }
    };

    const bool use = hist || bids;
    if (HASH && use && tid < nt) {
        note(0, n);
    }
    // the stream: by the threads that do not note, or by all
    const int  st    = HASH && use && nt < kLThreads ? tid - nt : tid;
    const int  sts   = HASH && use && nt < kLThreads ? kLThreads - nt : kLThreads;
    if (st < 0) {
    } else if constexpr (VEC) {
        const bool    wide = (reinterpret_cast<uintptr_t>(a.y) | (uintptr_t) a.ldo * sizeof(EO)) % 32 == 0;  // slices begin on 256 columns
        constexpr int U = 4, NI = 8 / vec16<TI>::N;
        for (int k0 = st * 8; k0 < n; k0 += U * sts * 8) {
            vec16<TI> in[U][NI];
            uint32_t  open[U];
#pragma unroll
            for (int u = 0; u < U; u++) {
                const int k = k0 + u * sts * 8;
                if (k < n) {
#pragma unroll
                    for (int q = 0; q < NI; q++) {
                        in[u][q].load(x + k + q * vec16<TI>::N);
                    }
                    open[u] = mask ? __ldg(mask + (k >> 5)) >> (k & 31) : 0xFFu;
                }
            }
#pragma unroll
            for (int u = 0; u < U; u++) {
                const int k = k0 + u * sts * 8;
                if (k < n) {
                    float v[8];
#pragma unroll
                    for (int j = 0; j < 8; j++) {
                        v[j] = (open[u] >> j) & 1u ? in[u][j / vec16<TI>::N].get(j % vec16<TI>::N) : -INFINITY;
                    }
                    store8<TO>(y + k, v, wide);
                }
            }
        }
    } else {
        constexpr int U = 8;
        for (int k0 = st; k0 < n; k0 += U * sts) {
            float v[U];
#pragma unroll
            for (int u = 0; u < U; u++) {
                const int k = k0 + u * sts;
                if (k < n) {
                    v[u] = io<TI>::to_f(x[k]);
                    v[u] = mask && !((__ldg(mask + (k >> 5)) >> (k & 31)) & 1u) ? -INFINITY : v[u];
                }
            }
#pragma unroll
            for (int u = 0; u < U; u++) {
                const int k = k0 + u * sts;
                if (k < n) {
                    y[k] = io<TO>::from_f(v[u]);
                }
            }
        }
    }
    if (use) {
        if constexpr (HASH) {
            __syncthreads();
            change(n_taken, [&](int i, int * k) {
                *k = (int) words[taken[i]];
                return words[a.slots + taken[i]];
            });
        } else {
            for (int k0 = 0; k0 < n; k0 += kWords) {
                const int k1 = min(n, k0 + kWords);
                __syncthreads();  // the part before has been read, the slice written
                note(k0, k1);
                __syncthreads();
                change(k1 - k0, [&](int i, int * k) {
                    *k = k0 + i;
                    return words[i];
                });
            }
        }
    }
    if (bad && a.err) {
        atomicOr(a.err, ACB_DEVERR_ID_RANGE);
    }
}

template <int TI, int TO> acb_status rules_launch(RulesArgs a, int rows, cudaStream_t st) {
    const bool vec  = (reinterpret_cast<uintptr_t>(a.x) | reinterpret_cast<uintptr_t>(a.y)) % 16 == 0 &&
                     (a.ld * type_size(TI) | a.ldo * type_size(TO)) % 16 == 0 && a.V % 8 == 0;
    const bool use  = a.r.hist || a.r.bias_ids;
    const bool hash = (a.r.hist ? a.r.hist_stride : 0) + (a.r.bias_ids ? a.r.n_bias : 0) <= kHashMost;
    // two blocks fit on an SM: one slice per block of a full GPU, or of four full GPUs where the rows alone fill it, and
    // at least 2048 columns each
    const int64_t full = 2 * (int64_t) num_sms();
    int64_t       cut  = rows * 2 > full ? (4 * full + rows - 1) / rows : full / rows;
    cut                = cut < 1 ? 1 : cut;
    int64_t slice      = ((a.V + cut - 1) / cut + 255) / 256 * 256;
    a.slice            = (int) (slice < 2048 ? 2048 : slice);
    // a long slice's stream takes longer than the history: four warps note while the others stream
    a.noters = a.slice >= 16384 && hash ? 128 : kLThreads;
    a.slots  = 64;
    a.shift  = 32 - 6;
    while (hash && a.slots / 4 * 3 < (a.r.hist ? a.r.hist_stride : 0) + (a.r.bias_ids ? a.r.n_bias : 0)) {
        a.slots *= 2;
        a.shift--;
    }
    const dim3   grid((unsigned) ((a.V + a.slice - 1) / a.slice), (unsigned) rows);
    const size_t smem = !use ? 0 : (hash ? 2 * a.slots : kWords) * sizeof(uint32_t);
    const auto   kern = vec ? (hash ? logits_rules_kernel<TI, TO, true, true> : logits_rules_kernel<TI, TO, true, false>)
                            : (hash ? logits_rules_kernel<TI, TO, false, true> : logits_rules_kernel<TI, TO, false, false>);
    if (smem) {
        // the kernel's limit, not this launch's size: it holds for the launches of every host thread
        const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int) (kWords * sizeof(uint32_t)));
        if (e != cudaSuccess) {
            set_last_cuda_error(e);
            return ACB_ERR_CUDA;
        }
    }
    kern<<<grid, kLThreads, smem, st>>>(a);
    return launch_status();
}

template <int TI> acb_status rules_launch(const RulesArgs & a, int to, int rows, cudaStream_t st) {
    return to == ACB_TYPE_F32   ? rules_launch<TI, ACB_TYPE_F32>(a, rows, st)
           : to == ACB_TYPE_F16 ? rules_launch<TI, ACB_TYPE_F16>(a, rows, st)
                                : rules_launch<TI, ACB_TYPE_BF16>(a, rows, st);
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
    const RulesArgs a  = { logits, ld, out, ld_out, V, r, err_flag, 0, 0, 0, 0 };
    cudaStream_t    st = (cudaStream_t) stream;
    return type == ACB_TYPE_F32   ? rules_launch<ACB_TYPE_F32>(a, out_type, rows, st)
           : type == ACB_TYPE_F16 ? rules_launch<ACB_TYPE_F16>(a, out_type, rows, st)
                                  : rules_launch<ACB_TYPE_BF16>(a, out_type, rows, st);
}
