// k_rope.cu -- rotary positions in every layout (acb_rope) and the table of angles for contexts longer than
// the trained one (acb_rope_table_scaled_host).
//
// With z = a + i b for a pair and w = c + i s its table entry, the rotation is z' = z w (w's conjugate for the
// inverse): 6 flops on 2 elements against a read and a write of both, so the memory bounds it. The vector form takes 16
// bytes at a time (with half pairs, 16 bytes of each half), a block one or more whole tokens, so that the angles of a token come
// from L1 for all its heads; where alignment or an odd width forbids that, it goes two elements at a time. 8191 tokens of 24
// heads of 192, bf16, 64 of them rotated as interleaved pairs: 29.6 us, 5.1 TB/s of 151 MB (a warp to a head, pair by
// pair: 86 us); threads for the next power of two of a token's vectors: 40 us. 4960 tokens of 29 heads of 110, f16, 66 of them
// rotated as half pairs: 31 us (a warp to a head 47).
#include <math.h>

#include <algorithm>
#include <type_traits>

#include "common.cuh"

namespace acb {
namespace {

struct RopeArgs {
    const void *    src;
    int64_t         sts, shs;
    void *          dst;
    int64_t         dts, dhs;
    int64_t         n_tok;
    int             n_heads, D, R;
    const int32_t * pos;
    const float *   table;
    int             max_pos;
    int *           err;
    bool            half, inverse, in_place;
};

// Units of two elements, the rotated pairs and then the pairs that are copied. threadIdx.x runs over a token's units (head by
// head), threadIdx.y over the block's tokens. WIDE: two neighbours are one aligned word.
template <int T, bool HALF, bool WIDE> __global__ void __launch_bounds__(256) rope_pair_kernel(const RopeArgs a, uint32_t units,
                                                                                                uint32_t magic) {
    using E         = typename io<T>::t;
    constexpr int U = 4;
    const int64_t t = (int64_t) blockIdx.x * blockDim.y + threadIdx.y;
    if (t >= a.n_tok) {
        return;
    }
    const int  p   = __ldg(a.pos + t);
    const bool bad = p < 0 || p >= a.max_pos;
    if (bad && threadIdx.x == 0 && a.err) {
        atomicOr(a.err, ACB_DEVERR_POS_RANGE);
    }
    const float *  w = a.table + (int64_t) (bad ? 0 : p) * a.R;
    const E *      x = reinterpret_cast<const E *>(a.src) + t * a.sts;
    E *            y = reinterpret_cast<E *>(a.dst) + t * a.dts;
    const uint32_t n = (uint32_t) a.n_heads * units;
    const int      rot = a.R / 2;
    union Two {
        E e[2];
        typename std::conditional<sizeof(E) == 2, uint32_t, uint2>::type word;
    };
    for (uint32_t i0 = threadIdx.x; i0 < n; i0 += U * blockDim.x) {
        Two      v[U];
        uint32_t h[U];
        int      u[U];
#pragma unroll
        for (int k = 0; k < U; k++) {  // all loads before any store
            const uint32_t i = i0 + k * blockDim.x;
            if (i < n) {
                h[k] = units == 1 ? i : __umulhi(i, magic);
                u[k] = (int) (i - h[k] * units);
                const E * q = x + (int64_t) h[k] * a.shs;
                if (HALF && u[k] < rot) {
                    v[k].e[0] = q[u[k]];
                    v[k].e[1] = q[u[k] + rot];
                } else if (WIDE) {
                    v[k].word = *reinterpret_cast<const decltype(v[k].word) *>(q + 2 * u[k]);
                } else {
                    v[k].e[0] = q[2 * u[k]];
                    v[k].e[1] = q[2 * u[k] + 1];
                }
            }
        }
#pragma unroll
        for (int k = 0; k < U; k++) {
            if (i0 + k * blockDim.x >= n) {
                break;
            }
            E * q = y + (int64_t) h[k] * a.dhs;
            if (bad) {
                v[k].e[0] = v[k].e[1] = io<T>::from_f(0.0f);
            } else if (u[k] < rot) {
                const float c = __ldg(w + 2 * u[k]), s0 = __ldg(w + 2 * u[k] + 1), s = a.inverse ? -s0 : s0;
                const float f = io<T>::to_f(v[k].e[0]), g = io<T>::to_f(v[k].e[1]);
                v[k].e[0]     = io<T>::from_f(__fsub_rn(__fmul_rn(f, c), __fmul_rn(g, s)));
                v[k].e[1]     = io<T>::from_f(__fadd_rn(__fmul_rn(f, s), __fmul_rn(g, c)));
            } else if (a.in_place) {
                continue;
            }
            if (HALF && u[k] < rot) {
                q[u[k]]       = v[k].e[0];
                q[u[k] + rot] = v[k].e[1];
            } else if (WIDE) {
                *reinterpret_cast<decltype(v[k].word) *>(q + 2 * u[k]) = v[k].word;
            } else {
                q[2 * u[k]]     = v[k].e[0];
                q[2 * u[k] + 1] = v[k].e[1];
            }
        }
    }
}

// Units of a head: half pairs, two 16-byte vectors R/2 apart; interleaved, one vector of whole pairs; then the vectors that are
// copied. threadIdx.x runs over a token's units (head by head), threadIdx.y over the block's tokens.
template <int T, bool HALF> __global__ void __launch_bounds__(256) rope_vec_kernel(const RopeArgs a, uint32_t rot_units,
                                                                                   uint32_t units, uint32_t magic) {
    using E           = typename io<T>::t;
    constexpr int V   = vec16<T>::N;
    const int64_t t   = (int64_t) blockIdx.x * blockDim.y + threadIdx.y;
    if (t >= a.n_tok) {
        return;
    }
    const int  p   = __ldg(a.pos + t);
    const bool bad = p < 0 || p >= a.max_pos;
    if (bad && threadIdx.x == 0 && a.err) {
        atomicOr(a.err, ACB_DEVERR_POS_RANGE);
    }
    const float *  w = a.table + (int64_t) (bad ? 0 : p) * a.R;
    const E *      x = reinterpret_cast<const E *>(a.src) + t * a.sts;
    E *            y = reinterpret_cast<E *>(a.dst) + t * a.dts;
    const uint32_t n = (uint32_t) a.n_heads * units;
    vec16<T>       lo[2], hi[2];
    auto           head_of = [&](uint32_t i) { return units == 1 ? i : __umulhi(i, magic); };
    auto           off_of  = [&](uint32_t u) { return u < rot_units ? (int) u * V : (HALF ? a.R : 0) + (int) (HALF ? u - rot_units : u) * V; };
    for (uint32_t i = threadIdx.x; i < n; i += 2 * blockDim.x) {
#pragma unroll
        for (int k = 0; k < 2; k++) {  // both units' loads before either's store
            const uint32_t j = i + k * blockDim.x;
            if (j < n) {
                const uint32_t h = head_of(j), u = j - h * units;
                const E *      q = x + (int64_t) h * a.shs + off_of(u);
                lo[k].load(q);
                if (HALF && u < rot_units) {
                    hi[k].load(q + a.R / 2);
                }
            }
        }
#pragma unroll
        for (int k = 0; k < 2; k++) {
            const uint32_t j = i + k * blockDim.x;
            if (j >= n) {
                break;
            }
            const uint32_t h = head_of(j), u = j - h * units;
            E *            q = y + (int64_t) h * a.dhs + off_of(u);
            if (bad) {
                lo[k].u = make_uint4(0, 0, 0, 0);
                hi[k].u = lo[k].u;
            } else if (u < rot_units) {
                const float4 * cs = reinterpret_cast<const float4 *>(w + (HALF ? 2 : 1) * V * u);
#pragma unroll
                for (int e = 0; e < (HALF ? V : V / 2); e += 2) {
                    const float4 c4 = __ldg(cs + e / 2);
#pragma unroll
                    for (int f = 0; f < 2; f++) {
                        const float c = f ? c4.z : c4.x, s0 = f ? c4.w : c4.y, sn = a.inverse ? -s0 : s0;
                        const int   ia = HALF ? e + f : 2 * (e + f);
                        const float g = lo[k].get(ia), z = HALF ? hi[k].get(ia) : lo[k].get(ia + 1);
                        const float r0 = __fsub_rn(__fmul_rn(g, c), __fmul_rn(z, sn));
                        const float r1 = __fadd_rn(__fmul_rn(g, sn), __fmul_rn(z, c));
                        lo[k].set(ia, r0);
                        if (HALF) {
                            hi[k].set(ia, r1);
                        } else {
                            lo[k].set(ia + 1, r1);
                        }
                    }
                }
            } else if (a.in_place) {
                continue;
            }
            lo[k].store(q);
            if (HALF && u < rot_units) {
                hi[k].store(q + a.R / 2);
            }
        }
    }
}

// whether every row of the call is made of whole aligned vectors
bool rope_vector(const RopeArgs & a, int type) {
    const int64_t v = 16 / type_size(type);
    const int64_t r = a.half ? a.R / 2 : a.R;
    return (reinterpret_cast<uintptr_t>(a.src) | reinterpret_cast<uintptr_t>(a.dst) | reinterpret_cast<uintptr_t>(a.table)) % 16 == 0 &&
           (a.sts | a.shs | a.dts | a.dhs) % v == 0 && a.D % v == 0 && r % v == 0 && a.R % 4 == 0;
}

template <int T> void rope_launch(const RopeArgs & a, cudaStream_t st) {
    constexpr int  V     = vec16<T>::N;
    const bool     vec   = rope_vector(a, T);
    const uint32_t rot   = (uint32_t) (a.half ? a.R / 2 : a.R) / V;
    const uint32_t units = vec ? rot + (uint32_t) (a.D - a.R) / V : (uint32_t) a.D / 2;
    const uint32_t n     = (uint32_t) a.n_heads * units;
    // i / units as the high word of i * magic: exact while i * units < 2^32 (2^14 heads of at most 2^9 units)
    const uint32_t magic = units == 1 ? 0 : (uint32_t) ((0x100000000ull + units - 1) / units);
    // Blocks of 256 threads, of vectors smaller ones where there are more than fit at once: 8191 tokens (24 heads of 192, bf16)
    // take 29.6 us in blocks of 64 and 32.3 in 256, 8 tokens (24 heads of 128, f32) 2.9 and 1.9. Each thread takes two vectors
    // or four pairs a turn, as few idle as whole warps allow; what a small token leaves of a block takes further tokens.
    uint32_t threads = 256;
    while (vec && threads > 64 && a.n_tok * std::min(threads, n) > (int64_t) 1024 * num_sms()) {
        threads /= 2;
    }
    const uint32_t each  = vec ? 2 : 4;
    const uint32_t turns = (n + threads * each - 1) / (threads * each);
    const uint32_t bx    = ((n + each * turns - 1) / (each * turns) + 31) / 32 * 32;
    const dim3     block(bx, threads / bx);
    const unsigned grid = (unsigned) ((a.n_tok + block.y - 1) / block.y);
    if (vec) {
        if (a.half) {
            rope_vec_kernel<T, true><<<grid, block, 0, st>>>(a, rot, units, magic);
        } else {
            rope_vec_kernel<T, false><<<grid, block, 0, st>>>(a, rot, units, magic);
        }
        return;
    }
    const int64_t two  = 2 * type_size(T);
    const bool    wide = (reinterpret_cast<uintptr_t>(a.src) | reinterpret_cast<uintptr_t>(a.dst)) % two == 0 &&
                      (a.sts | a.shs | a.dts | a.dhs) % 2 == 0;
    const auto kern = a.half ? (wide ? rope_pair_kernel<T, true, true> : rope_pair_kernel<T, true, false>)
                             : (wide ? rope_pair_kernel<T, false, true> : rope_pair_kernel<T, false, false>);
    kern<<<grid, block, 0, st>>>(a, units, magic);
}

}  // namespace
}  // namespace acb

using namespace acb;

extern "C" acb_status acb_rope(const void * src, int64_t src_tok_stride, int64_t src_head_stride, void * dst,
                               int64_t dst_tok_stride, int64_t dst_head_stride, int type, int64_t n_tok, int n_heads,
                               int head_dim, int rope_dim, int layout, const int32_t * pos, const float * rope_table,
                               int max_pos, int * err_flag, acb_stream_t stream) {
    if (!src || !dst || !pos || !rope_table || n_tok < 0 || n_heads <= 0 || max_pos <= 0 || src_tok_stride < 0 ||
        dst_tok_stride < 0 || src_head_stride < 0 || dst_head_stride < 0 || head_dim <= 0 || head_dim % 2 != 0 ||
        rope_dim < 2 || rope_dim > head_dim || rope_dim % 2 != 0 || layout < 0 || layout > 3) {
        return ACB_ERR_INVALID_ARG;
    }
    // one buffer in two layouts would be written before it is read
    const bool in_place = src == dst;
    if (in_place && (src_tok_stride != dst_tok_stride || src_head_stride != dst_head_stride)) {
        return ACB_ERR_INVALID_ARG;
    }
    // the destination's rows lie apart: tokens of heads or heads of tokens
    const bool    toks  = dst_tok_stride >= dst_head_stride;
    const int64_t inner = toks ? dst_head_stride : dst_tok_stride, outer = toks ? dst_tok_stride : dst_head_stride;
    const int64_t n_in = toks ? n_heads : n_tok, n_out = toks ? n_tok : n_heads;
    if ((n_in > 1 && inner < head_dim) || (n_out > 1 && outer < (n_in > 1 ? (n_in - 1) * inner : 0) + head_dim)) {
        return ACB_ERR_INVALID_ARG;
    }
    if (!is_io_type(type) || head_dim > 1024 || n_heads > 16384 || n_tok > (int64_t) INT32_MAX) {
        return ACB_ERR_UNSUPPORTED;
    }
    if (n_tok == 0) {
        return ACB_OK;
    }
    const RopeArgs a = { src,      src_tok_stride, src_head_stride, dst,        dst_tok_stride, dst_head_stride,
                         n_tok,    n_heads,        head_dim,        rope_dim,   pos,            rope_table,
                         max_pos,  err_flag,       (layout & ACB_ROPE_INTERLEAVED) == 0,
                         (layout & ACB_ROPE_INVERSE) != 0,          in_place };
    cudaStream_t st = (cudaStream_t) stream;
    if (type == ACB_TYPE_F32) {
        rope_launch<ACB_TYPE_F32>(a, st);
    } else if (type == ACB_TYPE_F16) {
        rope_launch<ACB_TYPE_F16>(a, st);
    } else {
        rope_launch<ACB_TYPE_BF16>(a, st);
    }
    return launch_status();
}

// Angles a_i = f_i p with f_i = base^(-2i/rope_dim) changed by the kind of scaling, all in double: a float angle of
// position 10^5 is off by up to 2^-7, a double one by 2^-36.
extern "C" acb_status acb_rope_table_scaled_host(float * table, int max_pos, int rope_dim, float base, int kind,
                                                 float factor, int orig_max_pos, float beta_fast, float beta_slow) {
    if (!table || max_pos <= 0 || rope_dim < 2 || rope_dim % 2 != 0 || !(base > 1.0f) || !isfinite(base) ||
        kind < ACB_ROPE_SCALE_NONE || kind > ACB_ROPE_SCALE_YARN || !(factor >= 1.0f) || !isfinite(factor)) {
        return ACB_ERR_INVALID_ARG;
    }
    if (kind == ACB_ROPE_SCALE_YARN &&
        (orig_max_pos <= 0 || !(beta_slow > 0.0f) || !(beta_fast > beta_slow) || !isfinite(beta_fast))) {
        return ACB_ERR_INVALID_ARG;
    }
    if (kind == ACB_ROPE_SCALE_NTK && rope_dim < 4) {
        return ACB_ERR_UNSUPPORTED;  // the exponent rope_dim / (rope_dim - 2) needs a second pair
    }
    const double pi2 = 6.283185307179586476925286766559;
    const int    n   = rope_dim / 2;
    double       b = base, mscale = 1.0;
    if (kind == ACB_ROPE_SCALE_NTK) {
        b *= pow((double) factor, (double) rope_dim / (rope_dim - 2));
    }
    double lo = 0.0, hi = 0.0;  // pair indices between which YaRN goes from unchanged to divided
    if (kind == ACB_ROPE_SCALE_YARN) {
        // the pair that turns r times over orig_max_pos: base^(-2i/rope_dim) orig_max_pos = 2 pi r
        auto pair_of = [&](double r) { return rope_dim * log(orig_max_pos / (r * pi2)) / (2.0 * log((double) base)); };
        lo           = fmax(0.0, floor(pair_of(beta_fast)));
        hi           = fmin((double) (rope_dim - 1), ceil(pair_of(beta_slow)));
        mscale       = 0.1 * log((double) factor) + 1.0;
    }
    for (int i = 0; i < n; i++) {
        double f = pow(b, -2.0 * i / rope_dim);
        if (kind == ACB_ROPE_SCALE_LINEAR) {
            f /= factor;
        } else if (kind == ACB_ROPE_SCALE_YARN) {
            const double t = fmin(1.0, fmax(0.0, (i - lo) / fmax(hi - lo, 1e-3)));
            f              = f * (1.0 - t) + f / factor * t;
        }
        for (int p = 0; p < max_pos; p++) {
            table[(int64_t) p * rope_dim + 2 * i]     = (float) (mscale * cos(f * p));
            table[(int64_t) p * rope_dim + 2 * i + 1] = (float) (mscale * sin(f * p));
        }
    }
    return ACB_OK;
}
