// k_attn_q4.cu -- causal attention over the paged 4-bit KV cache (acb_attn_kv_q4).
//
// One pass over the keys with the running reference m and sum l of the softmax. For the rows that share a kv head (its query
// heads times the sequence's new tokens) both products are matrix products on small tensor-core tiles:
//   S[key][row] = K[key][:] . Q[row][:]        A = keys as they are unpacked, B = queries
//   O[dim][row] += V^T[dim][key] P[key][row]   A = values, two keys to a register, B = P
// Every cached element is an f16 number (kv_q4.cuh), so A is exact; Q is scaled by a power of two per row into f16's range
// (an f32 query is the sum of two f16 numbers), and for an f32 output P goes in as the sum of two f16 numbers, so that both
// products carry 21 bits and more; for a 16-bit output P is one f16 number: half a step of 2^-11 of every weight, so at most 2^-11 of
// sum p |v|, next to the output's own rounding of 2^-8 (bf16: does not show) or 2^-11 (f16: 0.00023 against 64 bits where
// weights in f32 have 0.00021). Sums are f32, the weights' own of unrounded weights.
//
// Few rows have 1.125 bytes of cache per key and dimension against 4 flops a row, so the cache is read once: a warp takes 16 keys
// at a time and unpacks them into the registers that the tensor cores read -- the k index of a product may be any
// order of the dimensions as long as both operands agree, so a thread's share of a key is 16 consecutive bytes -- with the next tiles
// under way into the warp's own ring in shared memory. Long sequences are cut into chunks of keys, one block each; a second
// kernel joins the parts. 96 sequences of 200-8192 keys (32/8 heads of 128, bf16): 156 us, 3.0 TB/s of 468 MB; two of 131071
// (16/8 heads, f16): 97 us, 3.1 TB/s. The instructions bound it: 13 for 8 codes (a shift, four masks, eight f16
// operations), 208 of the 420 of a tile of 16 keys; issue slots are 71% busy, the integer pipe 64%.
#include <math.h>

#include <algorithm>
#include <type_traits>

#include "attn_q4.cuh"
#include "ptx.cuh"

namespace acb {
namespace {

constexpr int   kSplitWarps = 4;
constexpr int   kNoChunk    = 1 << 30;  // as many keys as a cache can have for one sequence
constexpr float kLag        = 8.0f;  // m follows a row's maximum when that has grown by more than 2^kLag
constexpr float kLift       = 6.0f;  // P is held times 2^kLift: at most 2^14, and whole f16 numbers down to 2^-20 of the maximum

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

__device__ __forceinline__ void mma16816(float * c, const uint32_t * a, uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

__device__ __forceinline__ uint32_t transpose8x8(uint32_t v) {
    uint32_t r;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
    return r;
}

// 16 keys and values of a warp in shared memory. With lane = 4 g + t a thread takes, of keys g and g + 8, the D/8 bytes from
// t D/8 on, and of values 2t, 2t+1, 2t+8, 2t+9 the D/16 bytes from g D/16 on: what the A operands of both products take. The
// pitches spread the lanes of every such access over all banks.
template <int D> struct Stage16 {
    static constexpr int KP = D == 256 ? 144 : D / 2, VP = D / 2 + 16;
    static constexpr int V = 16 * KP, KS = V + 16 * VP, VS = KS + D, BYTES = VS + D;
    static constexpr int KW = D / 32, VW = D / 64;

    // the copies of one warp, 16 bytes a lane: the rows of a tile are consecutive in the pool. What a lane copies and where to:
    const uint8_t * kc;
    const uint8_t * vc;
    const uint8_t * sc;
    uint32_t        kd, vd;

    __device__ __forceinline__ Stage16(const KvQ4 & kv, int lane)
        : kc(kv.kc + lane * 16), vc(kv.vc + lane * 16),
          sc(reinterpret_cast<const uint8_t *>(lane < D / 16 ? kv.ks : kv.vs) + lane % (D / 16) * 16),
          kd(lane / (D / 32) * KP + lane % (D / 32) * 16), vd(V + lane / (D / 32) * VP + lane % (D / 32) * 16) {}

    __device__ __forceinline__ void fill(uint32_t st, uint32_t row, int lane) const {
        const uint8_t * k = kc + (uint64_t) row * (D / 2);
        const uint8_t * v = vc + (uint64_t) row * (D / 2);
#pragma unroll
        for (int i = 0; i < D / 64; i++) {
            copy16(st + kd + i * (1024 / D) * KP, k + 512 * i);
            copy16(st + vd + i * (1024 / D) * VP, v + 512 * i);
        }
        if (lane < D / 8) {
            copy16(st + KS + lane * 16, sc + (uint64_t) row * (D / 16));
        }
    }
    static __device__ __forceinline__ void copy16(uint32_t dst, const void * src) {
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
    }
};

// where the parts of new token i of sequence s are, in rows of all heads
__device__ __forceinline__ int64_t part_row(const AttnQ4Args & a, int s, int i, int64_t tok) {
    return a.by_seq ? (int64_t) s * a.max_q + i : tok;
}

// dimension of nibble `hi` of byte b of a row's codes
__device__ __forceinline__ int dim_of(int b, int hi) {
    return (b >> 4) * 32 + (b & 15) + 16 * hi;
}

// blocks of an SM that the registers are held to
template <int T, int D, int NT> constexpr int kSplitBlocks = D == 256 || NT == 2 ? 2 : T == ACB_TYPE_F32 ? 4 : 5;

// tiles of a warp's ring
template <int D> constexpr int kStages = D == 256 ? 3 : 4;

// One block: up to 8 NT rows (r = new token * G + query head of the group) of one sequence and kv head, over one chunk of keys.
template <int T, int D, int NT>
__global__ void __launch_bounds__(32 * kSplitWarps, kSplitBlocks<T, D, NT>) attn_q4_split_kernel(const AttnQ4Args a) {
    constexpr int  KT  = D / 16;  // k steps of Q.K
    constexpr int  MT  = D / 16;  // 16-dimension tiles of the output
    constexpr int  QP  = T == ACB_TYPE_F32 ? 2 : 1;
    constexpr int  R   = 8 * NT;
    using T1           = typename io<T>::t;
    __shared__ int   s_hi[R], s_lo[R], s_first[R], s_last[R];  // of the rows: last and first key, and their chunks
    __shared__ float s_m[kSplitWarps][R], s_l[kSplitWarps][R], s_top[R];
    extern __shared__ __align__(16) uint8_t smem[];  // the warps' rings, then the sums of the warps' parts
    float (*s_o)[D + 4] = reinterpret_cast<float (*)[D + 4]>(smem);
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
    const int hk = blockIdx.y, s = blockIdx.z;
    const int rt = a.tiles == 1 ? 0 : blockIdx.x / a.n_split, split = blockIdx.x - rt * a.n_split;
    // new token of row r; the division only where there is more than one
    auto token_of = [&](int r) { return a.max_q == 1 ? (r >= a.G ? 1 : 0) : r / a.G; };
    ptx::grid_dep_launch();
    int64_t    row0;
    int        n, len;
    const bool ok = seq_bounds(a, s, &row0, &n, &len);
    if (!ok && a.err && threadIdx.x == 0) {
        atomicOr(a.err, ACB_DEVERR_LEN_RANGE);
    }
    const int r0 = rt * R;
    if (r0 >= n * a.G) {
        return;
    }
    // the keys that some row of this block sees
    const int i0 = token_of(r0), i1 = min(n - 1, token_of(r0 + R - 1));
    const int p0 = ok ? len - n + i0 : -1, p1 = ok ? len - n + i1 : -1;
    const int lo0 = a.window > 0 ? max(0, p0 - a.window + 1) : 0;
    // rows that see no key are written by the first block
    if (split == 0 && p0 < 0) {
        for (int e = threadIdx.x; e < R * D; e += 32 * kSplitWarps) {
            const int r = r0 + e / D, i = r / a.G;
            if (i < n && (!ok || len - n + i < 0) && row0 + i >= 0 && row0 + i < a.n_tok) {
                reinterpret_cast<T1 *>(a.o)[(row0 + i) * a.o_stride + (int64_t) (hk * a.G + r % a.G) * D + e % D] =
                    io<T>::from_f(0.0f);
            }
        }
    }
    const int c  = (lo0 > 0 ? lo0 / a.chunk : 0) + split;
    const int j0 = max(lo0, c * a.chunk), j1 = min(p1 + 1, (c + 1) * a.chunk);
    if (j0 >= j1) {
        return;
    }
    if (threadIdx.x < R) {
        const int i = token_of(r0 + threadIdx.x), p = i < n ? len - n + i : -1, lo = a.window > 0 ? max(0, p - a.window + 1) : 0;
        s_hi[threadIdx.x]    = p;
        s_lo[threadIdx.x]    = lo;
        s_first[threadIdx.x] = lo > 0 ? lo / a.chunk : 0;
        s_last[threadIdx.x]  = p >= 0 ? p / a.chunk : -1;
    }
    __syncthreads();
    // keys before full0 are behind the last row's window
    const int full0 = a.window > 0 ? max(0, p1 - a.window + 1) : 0;

    // queries: row g of each 8, the dimensions that meet this thread's bytes of a key
    uint32_t qf[QP][NT][KT][2];
    float    sc[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; nt++) {
        const int  r = r0 + nt * 8 + g, i = token_of(r);
        const T1 * q = reinterpret_cast<const T1 *>(a.q) + (row0 + i) * a.q_stride + (int64_t) (hk * a.G + r - i * a.G) * D;
        float      f[KT][4], mx = 0.0f;
#pragma unroll
        for (int w = 0; w < D / 64; w++) {
            // 8 bytes of codes are two runs of 8 dimensions: their low halves and their high halves
            const int b = t * (D / 8) + 8 * w;
            float     z[2][8];
#pragma unroll
            for (int h = 0; h < 2; h++) {
                const T1 * src = q + dim_of(b, h);
                if (i >= n) {
#pragma unroll
                    for (int e = 0; e < 8; e++) {
                        z[h][e] = 0.0f;
                    }
                } else if (a.q_vec) {
#pragma unroll
                    for (int v = 0; v < 8 / vec16<T>::N; v++) {
                        vec16<T> in;
                        in.load_nc(src + v * vec16<T>::N);
#pragma unroll
                        for (int e = 0; e < vec16<T>::N; e++) {
                            z[h][v * vec16<T>::N + e] = in.get(e);
                        }
                    }
                } else {
#pragma unroll
                    for (int e = 0; e < 8; e++) {
                        z[h][e] = io<T>::to_f(src[e]);
                    }
                }
            }
#pragma unroll
            for (int e = 0; e < 16; e++) {
                // order of unpack4 in a word: bytes 0 and 2 low, 0 and 2 high, 1 and 3 low, 1 and 3 high
                const float v                         = z[(e >> 1) & 1][4 * (e >> 3) + ((e >> 2) & 1) + 2 * (e & 1)];
                f[4 * w + 2 * (e >> 3) + ((e >> 2) & 1)][e & 3] = v;
                mx                                    = fmaxf(mx, fabsf(v));
            }
        }
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
        // 2^e with mx / 2^e in [1, 2): exponent field of mx, kept where 2^-e is a number
        int e = (int) (__float_as_uint(mx) >> 23);
        e     = mx == 0.0f || e == 255 ? 127 : min(max(e, 1), 253);
        // the scale's sign goes into the query: what is left is above 0, so that a masked score stays -inf
        const float down = a.scale_log2 == 0.0f ? 0.0f : copysignf(__uint_as_float((uint32_t) (254 - e) << 23), a.scale_log2);
        const float up   = __uint_as_float((uint32_t) e << 23);
#pragma unroll
        for (int k = 0; k < KT; k++) {
#pragma unroll
            for (int h = 0; h < 2; h++) {
                const float   x = f[k][2 * h] * down, y = f[k][2 * h + 1] * down;
                const __half2 hi = __floats2half2_rn(x, y);
                qf[0][nt][k][h]  = u32_of(hi);
                if (QP == 2) {
                    const float2 b          = __half22float2(hi);
                    qf[QP - 1][nt][k][h] = u32_of(__floats2half2_rn(x - b.x, y - b.y));
                }
            }
        }
        const float fs = fmaxf(fabsf(a.scale_log2) * up, 1.2e-38f);
        // scores come out with the row in the column index: rows 2t and 2t + 1, held by the lanes with g = 2t, 2t + 1
        sc[nt][0] = __shfl_sync(0xffffffffu, fs, 8 * t);
        sc[nt][1] = __shfl_sync(0xffffffffu, fs, 8 * t + 4);
    }

    // weights are 2^(score sc + lift); a score above thr makes lift follow (-inf: no key seen yet)
    float o[MT][NT][4], lift[NT][2], thr[NT][2], l[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; nt++) {
        lift[nt][0] = lift[nt][1] = 0.0f;
        thr[nt][0] = thr[nt][1] = -INFINITY;
        l[nt][0] = l[nt][1] = 0.0f;
#pragma unroll
        for (int mt = 0; mt < MT; mt++) {
            o[mt][nt][0] = o[mt][nt][1] = o[mt][nt][2] = o[mt][nt][3] = 0.0f;
        }
    }

    const int tb0    = (j0 & ~15) + 16 * warp;
    using St = Stage16<D>;
    constexpr int  STEP = 16 * kSplitWarps, NST = kStages<D>;
    const uint32_t ring = ptx::smem_u32(smem) + warp * (NST * St::BYTES);
    const uint8_t * mine = smem + warp * (NST * St::BYTES);
    const St        mover(a.kv, lane);

    // A tile; EDGE: one that some row does not see whole, with -inf for what it does not see and the values that no row sees
    // left out. The others, nearly all, have none of that in their code.
    auto take = [&](auto edge_tile, const int tb, const uint8_t * st) {
        constexpr bool EDGE = decltype(edge_tile)::value;
        // scores
        Words<St::KW>    k[2];
        const uint16_t * ksc = reinterpret_cast<const uint16_t *>(st + St::KS) + g * (D / 32) + t * D / 128;
        k[0].load_shared(st + g * St::KP + t * (D / 8));
        k[1].load_shared(st + (g + 8) * St::KP + t * (D / 8));
        float S[NT][4];
#pragma unroll
        for (int nt = 0; nt < NT; nt++) {
            S[nt][0] = S[nt][1] = S[nt][2] = S[nt][3] = 0.0f;
        }
#pragma unroll
        for (int w = 0; w < D / 32; w++) {
            uint32_t x[4], y[4];
            unpack4(k[0].w[w], __half2half2(__ushort_as_half(ksc[w / 4])), x);
            unpack4(k[1].w[w], __half2half2(__ushort_as_half(ksc[8 * (D / 32) + w / 4])), y);
            const uint32_t a0[4] = { x[0], y[0], x[1], y[1] }, a1[4] = { x[2], y[2], x[3], y[3] };
#pragma unroll
            for (int nt = 0; nt < NT; nt++) {
#pragma unroll
                for (int p = QP - 1; p >= 0; p--) {
                    mma16816(S[nt], a0, qf[p][nt][2 * w][0], qf[p][nt][2 * w][1]);
                    mma16816(S[nt], a1, qf[p][nt][2 * w + 1][0], qf[p][nt][2 * w + 1][1]);
                }
            }
        }
        if (EDGE) {
#pragma unroll
            for (int nt = 0; nt < NT; nt++) {
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const int j = tb + g + 8 * (e >> 1), r = nt * 8 + 2 * t + (e & 1);
                    if (j < max(j0, s_lo[r]) || j > min(j1 - 1, s_hi[r])) {
                        S[nt][e] = -INFINITY;
                    }
                }
            }
        }
        bool grow = false;
#pragma unroll
        for (int nt = 0; nt < NT; nt++) {
            grow = grow || fmaxf(S[nt][0], S[nt][2]) > thr[nt][0] || fmaxf(S[nt][1], S[nt][3]) > thr[nt][1];
        }
        if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
            for (int nt = 0; nt < NT; nt++) {
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    float x = fmaxf(S[nt][h], S[nt][h + 2]);
                    x       = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 4));
                    x       = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 8));
                    x       = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 16));
                    if (x > thr[nt][h]) {
                        const float to = kLift - x * sc[nt][h];
                        const float f  = thr[nt][h] == -INFINITY ? 1.0f : ex2(to - lift[nt][h]);
                        lift[nt][h]    = to;
                        thr[nt][h]     = x + kLag / sc[nt][h];
                        l[nt][h] *= f;
#pragma unroll
                        for (int mt = 0; mt < MT; mt++) {
                            o[mt][nt][h] *= f;
                            o[mt][nt][h + 2] *= f;
                        }
                    }
                }
            }
        }
        uint32_t ph[NT][2], pl[NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; nt++) {
#pragma unroll
            for (int h = 0; h < 2; h++) {
                const float x = ex2(fmaf(S[nt][2 * h], sc[nt][0], lift[nt][0]));
                const float y = ex2(fmaf(S[nt][2 * h + 1], sc[nt][1], lift[nt][1]));
                l[nt][0] += x;
                l[nt][1] += y;
                const __half2 hi = __floats2half2_rn(x, y);
                ph[nt][h]        = transpose8x8(u32_of(hi));
                if (QP == 2) {
                    const float2 b = __half22float2(hi);
                    pl[nt][h]      = transpose8x8(u32_of(__floats2half2_rn(x - b.x, y - b.y)));
                }
            }
        }
        Words<St::VW> v[4];
        uint16_t      vs[4];
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const int j = 2 * t + (i & 1) + (i & 2) * 4;
            v[i].load_shared(st + St::V + j * St::VP + g * (D / 16));
            vs[i] = reinterpret_cast<const uint16_t *>(st + St::VS)[j * (D / 32) + g * D / 256];
        }
        uint32_t vs01 = (uint32_t) vs[0] | ((uint32_t) vs[1] << 16);
        uint32_t vs23 = (uint32_t) vs[2] | ((uint32_t) vs[3] << 16);
        if (EDGE) {
            // a scale that is no number must not reach the rows that do not see its key (0 * NaN): it is taken out here and
            // put on the rows that do see it one by one
            uint32_t any = 0;
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const int j = tb + 2 * t + (i & 1) + (i & 2) * 4;
                if ((vs[i] & 0x7C00u) == 0x7C00u) {
                    (i < 2 ? vs01 : vs23) &= (i & 1) ? 0x0000FFFFu : 0xFFFF0000u;
                    any |= j >= j0 && j < j1;
                }
            }
            if (__any_sync(0xffffffffu, any)) {
                for (int j = max(tb, j0); j < min(tb + 16, j1); j++) {
                    const uint16_t d = reinterpret_cast<const uint16_t *>(st + St::VS)[(j - tb) * (D / 32) + g * D / 256];
                    if ((d & 0x7C00u) == 0x7C00u) {
#pragma unroll
                        for (int nt = 0; nt < NT; nt++) {
#pragma unroll
                            for (int h = 0; h < 2; h++) {
                                const int r = nt * 8 + 2 * t + h;
                                if (j >= s_lo[r] && j <= s_hi[r]) {
#pragma unroll
                                    for (int mt = 0; mt < MT; mt++) {
                                        o[mt][nt][h] = o[mt][nt][h + 2] = NAN;
                                    }
                                }
                            }
                        }
                    }
                }
            }
        }
#pragma unroll
        for (int w = 0; w < D / 64; w++) {
#pragma unroll
            for (int half = 0; half < 2; half++) {
                const uint32_t sel = half ? 0x7632u : 0x5410u;
                uint32_t       x[4], y[4];  // bytes 2 half, 2 half + 1: low, high, low, high nibble of two keys each
                unpack4(__byte_perm(v[0].w[w], v[1].w[w], sel), half2_of(vs01), x);
                unpack4(__byte_perm(v[2].w[w], v[3].w[w], sel), half2_of(vs23), y);
#pragma unroll
                for (int b = 0; b < 2; b++) {
                    const int      mt   = w * 4 + half * 2 + b;
                    const uint32_t f[4] = { x[2 * b], x[2 * b + 1], y[2 * b], y[2 * b + 1] };
#pragma unroll
                    for (int nt = 0; nt < NT; nt++) {
                        if (QP == 2) {
                            mma16816(o[mt][nt], f, pl[nt][0], pl[nt][1]);
                        }
                        mma16816(o[mt][nt], f, ph[nt][0], ph[nt][1]);
                    }
                }
            }
        }
    };
    // NST - 1 tiles under way in this warp's ring (registers for a tile ahead instead cost two fifths of the warps: 186 us for
    // the 96 sequences where this takes 159), the page of the next one looked up a turn before its copies
    int      pg   = tb0 < j1 ? a.kv.page_of(s, tb0) : 0;
    uint32_t lost = 0;  // bit of a stage: its page is not in the pool
    auto     fetch = [&](int tb, int slot) {
        if (tb < j1) {
            lost = (lost & ~(1u << slot)) | (uint32_t) (pg < 0) << slot;
            if (pg >= 0) {
                mover.fill(ring + slot * St::BYTES, a.kv.row(pg, hk, tb), lane);
            }
            if (tb + STEP < j1) {
                pg = a.kv.page_of(s, tb + STEP);
            }
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
#pragma unroll
    for (int i = 0; i < NST - 1; i++) {
        fetch(tb0 + i * STEP, i);
    }
    int slot = 0;
    for (int tb = tb0; tb < j1; tb += STEP) {
        asm volatile("cp.async.wait_group %0;" ::"n"(NST - 2) : "memory");
        __syncwarp();  // all lanes' copies of this stage are there, and all are done with the one that is filled next
        const int free = slot == 0 ? NST - 1 : slot - 1;
        fetch(tb + (NST - 1) * STEP, free);
        if ((lost >> slot) & 1u) {
            if (lane == 0 && a.err) {
                atomicOr(a.err, ACB_DEVERR_PAGE_RANGE);
            }
        } else {
            if (tb < full0 || tb < j0 || tb + 15 > p0 || tb + 15 >= j1) {
                take(std::true_type{}, tb, mine + slot * St::BYTES);
            } else {
                take(std::false_type{}, tb, mine + slot * St::BYTES);
            }
        }
        slot = slot == NST - 1 ? 0 : slot + 1;
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");

    // The four warps' parts, joined in the warps' order: each leaves its sums in shared memory as its registers hold them (value
    // v of lane x at 32 v + x), and then adds up a quarter of them.
    __syncthreads();  // the rings are done with
#pragma unroll
    for (int nt = 0; nt < NT; nt++) {
#pragma unroll
        for (int h = 0; h < 2; h++) {
            float x = l[nt][h];
            x += __shfl_xor_sync(0xffffffffu, x, 4);
            x += __shfl_xor_sync(0xffffffffu, x, 8);
            x += __shfl_xor_sync(0xffffffffu, x, 16);
            if (g == 0) {
                s_m[warp][nt * 8 + 2 * t + h] = thr[nt][h] == -INFINITY ? -INFINITY : -lift[nt][h];
                s_l[warp][nt * 8 + 2 * t + h] = x;
            }
        }
    }
    constexpr int NV   = MT * NT * 4;  // values of a lane
    float *       part = reinterpret_cast<float *>(smem);
#pragma unroll
    for (int v = 0; v < NV; v++) {
        part[(warp * NV + v) * 32 + lane] = o[v / (4 * NT)][v / 4 % NT][v % 4];
    }
    __syncthreads();
    // what each warp's sums are taken by, and the rows' sums of weights
    if (threadIdx.x < R) {
        const int   r = threadIdx.x;
        const float M = fmaxf(fmaxf(s_m[0][r], s_m[1][r]), fmaxf(s_m[2][r], s_m[3][r]));
        float       L = 0.0f;
#pragma unroll
        for (int w = 0; w < kSplitWarps; w++) {
            const float f = s_m[w][r] == -INFINITY ? 0.0f : ex2(s_m[w][r] - M);
            L += s_l[w][r] * f;
            s_m[w][r] = f;
        }
        s_top[r] = M;
        s_l[0][r] = L;
    }
    __syncthreads();
    float sum[NV / kSplitWarps];
#pragma unroll
    for (int k = 0; k < NV / kSplitWarps; k++) {
        const int v = warp * (NV / kSplitWarps) + k, r = (v / 4 % NT) * 8 + 2 * t + (v & 1);
        sum[k]      = 0.0f;
#pragma unroll
        for (int w = 0; w < kSplitWarps; w++) {
            sum[k] += part[(w * NV + v) * 32 + lane] * s_m[w][r];
        }
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < NV / kSplitWarps; k++) {
        const int v = warp * (NV / kSplitWarps) + k, r = (v / 4 % NT) * 8 + 2 * t + (v & 1);
        s_o[r][dim_of(g * (D / 16) + v / (4 * NT), (v >> 1) & 1)] = sum[k];
    }
    __syncthreads();
    for (int e = threadIdx.x; e < R * D / 4; e += 32 * kSplitWarps) {
        const int rr = e / (D / 4), d = (e % (D / 4)) * 4;
        const int r = r0 + rr, i = token_of(r), c0 = s_first[rr], c1 = s_last[rr];
        if (c < c0 || c > c1) {  // no key of this row in this chunk (or no such row)
            continue;
        }
        const float   L   = s_l[0][rr];
        const float4  v   = *reinterpret_cast<const float4 *>(&s_o[rr][d]);
        const int64_t tok = row0 + i;
        const int     h   = hk * a.G + r - i * a.G;
        if (c0 == c1) {  // every key of this row was in this chunk
            const float inv = L != 0.0f ? 1.0f / L : 0.0f;
            T1 *        y   = reinterpret_cast<T1 *>(a.o) + tok * a.o_stride + (int64_t) h * D + d;
            y[0]            = io<T>::from_f(v.x * inv);
            y[1]            = io<T>::from_f(v.y * inv);
            y[2]            = io<T>::from_f(v.z * inv);
            y[3]            = io<T>::from_f(v.w * inv);
        } else {
            const int64_t slot = (part_row(a, s, i, tok) * a.Nh + h) * a.n_split + c % a.n_split;
            *reinterpret_cast<float4 *>(a.part_o + slot * D + d) = v;
            if (d == 0) {
                a.part_ml[slot] = make_float2(s_top[rr], L);
            }
        }
    }
}

// Joins the chunks of a row that had more than one: a block per row, the chunks dealt to its warps (the loads of one warp
// follow each other, those of several do not wait: 108 chunks took some 60 us with one warp a row), the warps' sums added in
// their order.
constexpr int kJoinWarps = 4;

template <int T, int D> __global__ void __launch_bounds__(32 * kJoinWarps) attn_q4_join_kernel(const AttnQ4Args a) {
    constexpr int    E = D / 32;
    using T1           = typename io<T>::t;
    __shared__ float s_l[kJoinWarps], s_o[kJoinWarps][D];
    const int        lane = threadIdx.x & 31, warp = threadIdx.x >> 5, hk = blockIdx.y, s = blockIdx.z, r = blockIdx.x;
    ptx::grid_dep_wait();
    int64_t    row0;
    int        n, len;
    const bool ok = seq_bounds(a, s, &row0, &n, &len);
    const int  i = a.max_q == 1 ? 0 : r / a.G, p = len - n + i;
    if (!ok || i >= n || p < 0) {
        return;
    }
    const int c0 = (a.window > 0 ? max(0, p - a.window + 1) : 0) / a.chunk, c1 = p / a.chunk;
    if (c0 == c1) {
        return;
    }
    const int64_t tok = row0 + i;
    const int     h   = hk * a.G + r - i * a.G;
    const int64_t at  = (part_row(a, s, i, tok) * a.Nh + h) * a.n_split;
    float         M = -INFINITY, L = 0.0f, o[E];
    for (int c = c0 + lane; c <= c1; c += 32) {
        M = fmaxf(M, a.part_ml[at + c % a.n_split].x);
    }
    M = warp_max(M);
#pragma unroll
    for (int e = 0; e < E; e++) {
        o[e] = 0.0f;
    }
#pragma unroll 4
    for (int c = c0 + warp; c <= c1; c += kJoinWarps) {
        const int64_t slot = at + c % a.n_split;
        const float2  ml   = a.part_ml[slot];
        const float   f    = M == -INFINITY ? 1.0f : ex2(ml.x - M);
        L += ml.y * f;
#pragma unroll
        for (int e = 0; e < E; e++) {
            o[e] += a.part_o[slot * D + e * 32 + lane] * f;
        }
    }
#pragma unroll
    for (int e = 0; e < E; e++) {
        s_o[warp][e * 32 + lane] = o[e];
    }
    if (lane == 0) {
        s_l[warp] = L;
    }
    __syncthreads();
    L               = (s_l[0] + s_l[1]) + (s_l[2] + s_l[3]);
    const float inv = L != 0.0f ? 1.0f / L : 0.0f;
    T1 *        y   = reinterpret_cast<T1 *>(a.o) + tok * a.o_stride + (int64_t) h * D;
    for (int d = threadIdx.x; d < D; d += 32 * kJoinWarps) {
        y[d] = io<T>::from_f(((s_o[0][d] + s_o[1][d]) + (s_o[2][d] + s_o[3][d])) * inv);
    }
}

using Kernel = void (*)(const AttnQ4Args);

template <int T, int NT> Kernel split_kernel(int D) {
    return D == 64 ? attn_q4_split_kernel<T, 64, NT> : D == 128 ? attn_q4_split_kernel<T, 128, NT>
                                                                : attn_q4_split_kernel<T, 256, NT>;
}

template <int T> Kernel split_kernel(int D, int nt) {
    return nt == 1 ? split_kernel<T, 1>(D) : D == 64 ? attn_q4_split_kernel<T, 64, 2> : attn_q4_split_kernel<T, 128, 2>;
}

template <int T> Kernel join_kernel(int D) {
    return D == 64 ? attn_q4_join_kernel<T, 64> : D == 128 ? attn_q4_join_kernel<T, 128> : attn_q4_join_kernel<T, 256>;
}

// How the keys are cut. Rows of one kv head in tiles of 8 or 16 (8 for heads of 256, whose sums fill the registers); chunks
// of a multiple of 64 keys (four warps of 16), as many as fill the GPU, but none below 256 keys: a chunk's part costs its rows
// 4 (D + 2) bytes twice, against 1.125 D bytes a key. A call of so few rows and heads that 256 keys a block would leave
// most SMs idle goes down to 128 (one sequence of 1536 keys, 8 kv heads: 10.1 us at 256, 8.9 at 128; 24 sequences of up to
// 4000 with drafts: 15.2 at 256, 19.5 at 128).

struct Plan {
    int     nt, tiles, chunk, n_split;
    int64_t most;  // n_split of any window at these sizes is at most this
    int64_t rows;  // up to so many rows of a sequence and kv head nt and most stay as they are
};

Plan make_plan(const acb_kv_q4 * kv, int n_heads, int max_q, int max_kv, int window) {
    Plan          p;
    const int64_t rows   = (int64_t) max_q * (n_heads / kv->n_kv_heads);
    p.nt                 = rows <= 8 || kv->head_dim == 256 ? 1 : 2;
    p.tiles              = (int) ((rows + 8 * p.nt - 1) / (8 * p.nt));
    const int64_t keys   = window > 0 && (int64_t) window + max_q < max_kv ? (int64_t) window + max_q : max_kv;
    const int64_t tasks  = (int64_t) p.tiles * kv->n_kv_heads * kv->n_seq;
    // One part per block of a full GPU where that cuts each sequence's keys at least four times; otherwise the parts of
    // sequences of very different lengths are to even out, so six times as many. (96 sequences of 200-8192 keys: 185 us at
    // three times, 159 at six. Two of 131071, before the warps were joined as now: 124 us at 111 parts each, 142 at 185, 180 at
    // 296.)
    const int64_t slots  = (int64_t) num_sms() * 5;
    const int64_t parts  = slots / tasks >= 4 ? slots : 6 * slots;
    const int64_t splits = parts / tasks;
    const int64_t least  = tasks * 4 <= num_sms() ? 128 : 256;
    const int64_t cuts   = (max_kv + least - 1) / least;
    if (splits <= 1 || cuts <= 1) {  // and so it is for any more rows
        p.n_split = 1;
        p.most    = 1;
        p.chunk   = kNoChunk;
        p.rows    = INT64_MAX;
        return p;
    }
    // The most tasks that give as many splits. (Where parts is slots these are 4 or more, so it is slots for those tasks too.)
    int64_t same = parts / splits;
    if (least == 128 && same > num_sms() / 4) {
        same = num_sms() / 4;
    }
    p.rows = p.nt == 1 && kv->head_dim != 256 ? 8 : same / ((int64_t) kv->n_kv_heads * kv->n_seq) * (8 * p.nt);
    int64_t chunk = (keys + splits - 1) / splits;
    chunk         = ((chunk < least ? least : chunk) + 63) / 64 * 64;
    p.chunk       = (int) chunk;
    // a window's keys can begin anywhere in a chunk
    p.n_split = (int) ((keys + chunk - 1) / chunk) + (keys < max_kv ? 1 : 0);
    p.most    = (splits < cuts ? splits : cuts) + 1;
    return p;
}

// Tokens that can have parts: a batch may be padded with rows that belong to no sequence, and then there are at most so many.
int64_t part_rows(const acb_kv_q4 * kv, int64_t n_tok, int64_t max_q) {
    return std::min<int64_t>(n_tok, max_q * kv->n_seq);
}

size_t plan_bytes(int64_t n_split, const acb_kv_q4 * kv, int64_t rows, int n_heads) {
    return n_split <= 1 ? 0 : (size_t) rows * n_heads * n_split * (kv->head_dim + 2) * sizeof(float);
}

}  // namespace
}  // namespace acb

using namespace acb;

extern "C" size_t acb_attn_kv_q4_work_bytes(const acb_kv_q4 * kv, int64_t n_tok, int n_heads, int max_q_len,
                                            int max_kv_len) {
    KvQ4 d;
    if (kv_q4_check(kv, &d) != ACB_OK || n_tok <= 0 || n_heads <= 0 || n_heads % kv->n_kv_heads != 0 || max_q_len <= 0 ||
        max_kv_len <= 0) {
        return 0;
    }
    // Enough for every call of at most these sizes. Fewer rows a sequence can mean more chunks or fewer (make_plan's rule has a
    // step), so every count of chunks that they can have is asked, with the most rows that have it.
    const int64_t G    = n_heads / kv->n_kv_heads;
    size_t        most = 0;
    for (int64_t q = 1; q <= max_q_len; q++) {
        const Plan p       = make_plan(kv, n_heads, (int) q, max_kv_len, 0);
        q                  = std::min<int64_t>(max_q_len, p.rows / G);
        const size_t bytes = plan_bytes(p.most, kv, part_rows(kv, n_tok, q), n_heads);
        most                = bytes > most ? bytes : most;
    }
    return most;
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
        max_kv_len < 0 || window < 0 || !isfinite(scale) || q_stride < (int64_t) n_heads * kv->head_dim ||
        o_stride < (int64_t) n_heads * kv->head_dim || (!q_start && (n_tok != kv->n_seq || max_q_len != 1)) ||
        (work && !kv_q4_aligned(work))) {
        return ACB_ERR_INVALID_ARG;
    }
    if (max_kv_len > (int64_t) kv->max_pages * kv->page_size) {
        return ACB_ERR_OUT_OF_RANGE;
    }
    if (!is_io_type(type) || kv->n_kv_heads > 65535 || kv->n_seq > 65535 ||
        (int64_t) max_q_len * n_heads > (1 << 24)) {
        return ACB_ERR_UNSUPPORTED;
    }
    if (q == o && n_tok > 1 && q_stride != o_stride) {
        return ACB_ERR_INVALID_ARG;  // one buffer in two layouts would be written before it is read
    }
    if (n_tok == 0) {
        return ACB_OK;
    }
    // A window of all keys is none. What is left is far from where a position less a window leaves 32 bits.
    window             = window >= max_kv_len ? 0 : window;
    Plan          p    = make_plan(kv, n_heads, max_q_len, max_kv_len, window);
    const int64_t rows = part_rows(kv, n_tok, max_q_len);
    if (p.n_split > 1 && (!work || work_bytes < plan_bytes(p.n_split, kv, rows, n_heads))) {
        p.n_split = 1;
        p.chunk   = kNoChunk;
    }
    a.q          = q;
    a.q_stride   = q_stride;
    a.n_tok      = n_tok;
    a.Nh         = n_heads;
    a.G          = n_heads / kv->n_kv_heads;
    a.q_start    = q_start;
    a.kv_len     = kv_len;
    a.max_q      = max_q_len;
    a.max_kv     = max_kv_len;
    a.window     = window;
    a.scale_log2 = scale * 1.4426950408889634f;
    a.o          = o;
    a.o_stride   = o_stride;
    a.err        = err_flag;
    a.q_vec      = reinterpret_cast<uintptr_t>(q) % 16 == 0 && q_stride * type_size(type) % 16 == 0;
    a.chunk      = p.chunk;
    a.n_split    = p.n_split;
    a.tiles      = p.tiles;
    const int D  = kv->head_dim;
    // the sums first: their rows are whole multiples of 16 bytes, whatever the number of parts
    a.part_o     = reinterpret_cast<float *>(work);
    a.part_ml    = reinterpret_cast<float2 *>(a.part_o + rows * n_heads * p.n_split * D);
    a.rows       = rows;
    a.by_seq     = rows < n_tok;
    if (attn_q4_tc_wanted(a, type, D)) {
        return attn_q4_tc_launch(a, type, D, (cudaStream_t) stream);
    }
    const Kernel kern = type == ACB_TYPE_F32   ? split_kernel<ACB_TYPE_F32>(D, p.nt)
                        : type == ACB_TYPE_F16 ? split_kernel<ACB_TYPE_F16>(D, p.nt)
                                               : split_kernel<ACB_TYPE_BF16>(D, p.nt);
    const size_t smem = (size_t) kSplitWarps * (D == 64 ? kStages<64> * Stage16<64>::BYTES : D == 128 ? kStages<128> * Stage16<128>::BYTES
                                                                                                : kStages<256> * Stage16<256>::BYTES);
    const cudaError_t ea = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int) smem);
    if (ea != cudaSuccess) {
        set_last_cuda_error(ea);
        return ACB_ERR_CUDA;
    }
    kern<<<dim3((unsigned) (p.tiles * p.n_split), (unsigned) kv->n_kv_heads, (unsigned) kv->n_seq), 32 * kSplitWarps, smem,
           (cudaStream_t) stream>>>(a);
    const acb_status st = launch_status();
    if (st != ACB_OK || p.n_split == 1) {
        return st;
    }
    const Kernel join = type == ACB_TYPE_F32   ? join_kernel<ACB_TYPE_F32>(D)
                        : type == ACB_TYPE_F16 ? join_kernel<ACB_TYPE_F16>(D)
                                               : join_kernel<ACB_TYPE_BF16>(D);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim            = dim3((unsigned) (max_q_len * a.G), (unsigned) kv->n_kv_heads, (unsigned) kv->n_seq);
    cfg.blockDim           = dim3(32 * kJoinWarps);
    cfg.stream             = (cudaStream_t) stream;
    cudaLaunchAttribute attr[1];
    attr[0].id                                         = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs                                          = attr;
    cfg.numAttrs                                       = 1;
    const cudaError_t e                                = cudaLaunchKernelEx(&cfg, join, a);
    if (e != cudaSuccess) {
        set_last_cuda_error(e);
        return ACB_ERR_CUDA;
    }
    return ACB_OK;
}
