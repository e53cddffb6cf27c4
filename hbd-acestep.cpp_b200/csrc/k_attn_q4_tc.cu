// k_attn_q4_tc.cu -- attention over the paged 4-bit KV cache for chunks of prompts, on the 5th-generation tensor cores.
//
// One CTA per 128 rows (new token * G + query head of the group) of a sequence and kv head; key blocks of 128. The layout of
// TMEM and the softmax are those of k_attn_tc.cu: two S/P buffers, O and Q in TMEM, A of both products from TMEM, two softmax
// threads a row. What differs is where K and V come from: four warps read the codes from the pages and write f16 tiles
// into shared memory (every cached value is an f16 number, so nothing is rounded), K^ [key][dim] and V^T [dim][key], both
// K-major with the 128-byte swizzle:
//   K: a thread a key; the 8 dimensions of a word of codes make one 16-byte unit in the order that unpack4 gives them, and Q
//      is put into TMEM in the same order (a product does not depend on the order of its k index);
//   V: a thread 8 keys by 16 dimensions: the words of two keys are merged by halves, so that unpack4 gives pairs of keys, and
//      four pairs make the 16-byte unit of a dimension.
// A block costs the tensor cores 2 x 512 cycles (D = 128), the exponentials 1024 cycles of the special-function units, and the
// unpacking about 520 issue slots of each scheduler beside the softmax's 700: all three overlap.
//
// Every wait is bounded, as in k_attn_tc.cu.
#include "attn_q4.cuh"
#include "ptx.cuh"
#include "tc.cuh"

namespace acb {
namespace {

constexpr int   kQtRows    = 128;
constexpr int   kQtKeys    = 128;
constexpr int   kQtSoft    = 8;   // softmax warps 0..7
constexpr int   kQtMma     = 8;   // the warp that issues the products
constexpr int   kQtUnpack  = 4;   // unpacking warps 9..12
constexpr int   kQtThreads = 32 * (kQtSoft + 1 + kQtUnpack);
constexpr float kQtLag     = 8.0f;  // the reference maximum moves when exceeded by more than 2^kQtLag
constexpr float kQtLift    = 6.0f;  // P is held times 2^kQtLift: at most 2^14
constexpr int   kQtRing    = 8;     // blocks whose notes are kept

template <int D> struct QtLayout {
    static constexpr int KB = kQtKeys * D * 2, VB = kQtKeys * D * 2, NK = 2, NV = 2;
    static constexpr int TOTAL = NK * KB + NV * VB;
    // TMEM columns: S/P buffers at 0 and 128, O at 256, Q at 384 (two f16 a column)
    static constexpr uint32_t TO = 256, TQ = 384;
};

template <int T, int D, bool ALIGNED> __global__ void __launch_bounds__(kQtThreads, 1) attn_q4_tc_kernel(const AttnQ4Args a) {
    using Lay = QtLayout<D>;
    using T1  = typename io<T>::t;
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    uint8_t *  sK      = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint8_t *  sV      = sK + Lay::NK * Lay::KB;
    uint64_t * q_full  = reinterpret_cast<uint64_t *>(sV + Lay::NV * Lay::VB);
    uint64_t * k_full  = q_full + 1;
    uint64_t * k_empty = k_full + Lay::NK;
    uint64_t * v_full  = k_empty + Lay::NK;
    uint64_t * v_empty = v_full + Lay::NV;
    uint64_t * s_full  = v_empty + Lay::NV;  // [2]
    uint64_t * p_full  = s_full + 2;         // [2]
    uint64_t * pv_done = p_full + 2;         // [2]
    uint64_t * o_done  = pv_done + 2;
    uint64_t * xbar    = o_done + 1;  // [4]: softmax pairs, one per TMEM lane quarter
    uint32_t * tmem_slot = reinterpret_cast<uint32_t *>(xbar + 4);
    __shared__ volatile int abort_flag;
    __shared__ float        xchg[2 * 2 * kQtRows];  // [parity][half][row]
    // notes on a block, for what hardly ever happens: keys whose page is not in the pool, and per 32 dimensions the keys whose
    // value scale is no number (their values are left out of the product, where 0 * NaN would reach the rows that do not see
    // them, and make their dimensions NaN in the rows that do)
    __shared__ uint32_t bad_key[kQtRing][4], bad_val[kQtRing][D / 32][4];
    __shared__ int      bad_any[kQtRing][2];

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int hk = blockIdx.y, s = blockIdx.z;
    int64_t    row0;
    int        n, len;
    const bool okay = seq_bounds(a, s, &row0, &n, &len);
    if (!okay && a.err && threadIdx.x == 0) {
        atomicOr(a.err, ACB_DEVERR_LEN_RANGE);
    }
    // the longest rows first: what is left for the end is short
    const int r0 = (int) (gridDim.x - 1 - blockIdx.x) * kQtRows;
    if (r0 >= n * a.G) {
        return;
    }
    const int i0 = r0 / a.G, i1 = min(n - 1, (r0 + kQtRows - 1) / a.G);
    const int p0 = okay ? len - n + i0 : -1, p1 = okay ? len - n + i1 : -1;
    const int key_lo = a.window > 0 ? max(0, p0 - a.window + 1) : 0;
    const int kb_lo  = key_lo / kQtKeys;
    const int nblk   = p1 < 0 ? 0 : p1 / kQtKeys + 1 - kb_lo;

    if (threadIdx.x == 0) {
        abort_flag = 0;
        ptx::mbar_init(q_full, kQtSoft);
        for (int i = 0; i < Lay::NK; i++) {
            ptx::mbar_init(&k_full[i], kQtUnpack);
            ptx::mbar_init(&k_empty[i], 1);
        }
        for (int i = 0; i < Lay::NV; i++) {
            ptx::mbar_init(&v_full[i], kQtUnpack);
            ptx::mbar_init(&v_empty[i], 1);
        }
        for (int i = 0; i < 2; i++) {
            ptx::mbar_init(&s_full[i], 1);
            ptx::mbar_init(&p_full[i], kQtSoft);
            ptx::mbar_init(&pv_done[i], 1);
        }
        ptx::mbar_init(o_done, 1);
        for (int x = 0; x < 4; x++) {
            ptx::mbar_init(&xbar[x], 2);
        }
        ptx::fence_mbar_init();
    }
    for (int i = threadIdx.x; i < kQtRing * 4; i += kQtThreads) {
        (&bad_key[0][0])[i] = 0;
    }
    for (int i = threadIdx.x; i < kQtRing * (D / 32) * 4; i += kQtThreads) {
        (&bad_val[0][0][0])[i] = 0;
    }
    if (threadIdx.x < kQtRing * 2) {
        (&bad_any[0][0])[threadIdx.x] = 0;
    }
    if (warp == kQtMma) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(ptx::smem_u32(tmem_slot)),
                     "r"(512));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    const uint32_t tO = tmem + Lay::TO, tQ = tmem + Lay::TQ;

    if (warp > kQtMma) {
        // ---- unpacking ----
        const int tid = threadIdx.x - 32 * (kQtMma + 1);  // 0..127
        // K: this thread's key of a block
        Words<D / 8>  kw;
        Words<D / 64> ksw;
        int           kpg = 0;
        auto          key_of = [&](int i) { return min((kb_lo + i) * kQtKeys + tid, p1); };
        auto          k_page = [&](int i) { kpg = a.kv.page_of(s, key_of(i)); };
        bool          k_bad  = false;
        auto          k_load = [&](int i) {
            const int j = key_of(i);
            k_bad       = kpg < 0;
            if (!k_bad) {
                const int64_t row = a.kv.row(kpg, hk, j);
                kw.load(a.kv.kc + row * (D / 2));
                ksw.load(a.kv.ks + row * (D / 32));
            }
        };
        // V: 8 keys from 8 kg on, 16 dimensions: the 8 bytes from 8 wq on; lanes of a store phase differ in kg
        const int kg = (tid & 7) | ((tid >> 6) << 3), wq = (tid >> 3) & 7;
        constexpr bool ALL = D == 128;  // heads of 64 have 4 such 8-byte runs: half the threads have none
        const bool     v_on = ALL || wq < 4;
        uint2          vw[8];
        uint16_t       vs[8];
        int            vpg = 0;
        uint32_t       v_bad = 0;
        auto           v_page = [&](int i) { vpg = a.kv.page_of(s, min((kb_lo + i) * kQtKeys + 8 * kg, p1)); };
        auto           v_load = [&](int i) {
            const int j = (kb_lo + i) * kQtKeys + 8 * kg;  // 8 keys of one page (pages hold 16 or more)
            if (v_on) {
                const int64_t   row = vpg < 0 ? 0 : a.kv.row(vpg, hk, j);
                const uint8_t * c   = a.kv.vc + row * (D / 2) + wq * 8;
                const uint16_t * d  = a.kv.vs + row * (D / 32) + (wq >> 1);
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    // a key past the last one: none of its own (the page may hold anything there)
                    const bool in = vpg >= 0 && j + e <= p1;
                    vw[e]         = in ? __ldg(reinterpret_cast<const uint2 *>(c + e * (D / 2))) : make_uint2(0, 0);
                    vs[e]         = in ? __ldg(d + e * (D / 32)) : (uint16_t) 0;
                }
            }
        };
        if (nblk > 0) {
            k_page(0);
            v_page(0);
            k_load(0);
        }
        for (int i = 0; i < nblk; i++) {
            v_load(i);
            if (i + 1 < nblk) {
                k_page(i + 1);
                v_page(i + 1);
            }
            const int sk = i % Lay::NK, sv = i % Lay::NV, note = i % kQtRing;
            if (!__all_sync(0xffffffffu, i < Lay::NK || tc_wait(&k_empty[sk], (i / Lay::NK - 1) & 1, &abort_flag, a.err))) {
                break;
            }
            // Room for the notes of block i + 2, where those of block i - 6 are: S(i - 2) is done, so the softmax has published
            // P(i - 4) and looked at block i - 6; and no unpacking warp is at block i + 2 before this one has filled block i.
            if (tid < 32) {
                const int next = (i + 2) % kQtRing;
                if (lane < 4) {
                    bad_key[next][lane] = 0;
                }
                if (lane < (D / 32) * 4) {
                    (&bad_val[next][0][0])[lane] = 0;
                }
                if (lane < 2) {
                    bad_any[next][lane] = 0;
                }
            }
            {
                const bool gone = (kb_lo + i) * kQtKeys + tid > p1;
                if (k_bad && !gone) {
                    atomicOr(&bad_key[note][tid >> 5], 1u << (tid & 31));
                    bad_any[note][0] = 1;
                    if (a.err) {
                        atomicOr(a.err, ACB_DEVERR_PAGE_RANGE);
                    }
                }
                uint8_t * dst = sK + sk * Lay::KB + tid * 128;
#pragma unroll
                for (int w = 0; w < D / 8; w++) {
                    const uint32_t sc = ksw.w[w / 8] >> (16 * ((w / 4) & 1));
                    uint32_t       r[4];
                    unpack4(kw.w[w], __half2half2(__ushort_as_half((uint16_t) (k_bad || gone ? 0u : sc))), r);
                    *reinterpret_cast<uint4 *>(dst + (w / 8) * 16384 + (((w & 7) ^ (tid & 7)) << 4)) = make_uint4(r[0], r[1], r[2], r[3]);
                }
            }
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) {
                ptx::mbar_arrive(&k_full[sk]);
            }
            if (i + 1 < nblk) {
                k_load(i + 1);
            }
            if (!__all_sync(0xffffffffu, i < Lay::NV || tc_wait(&v_empty[sv], (i / Lay::NV - 1) & 1, &abort_flag, a.err))) {
                break;
            }
            if (v_on) {
                v_bad = 0;
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    if ((vs[e] & 0x7C00u) == 0x7C00u) {
                        vs[e] = 0;
                        v_bad |= 1u << e;
                    }
                }
                if (v_bad) {
                    atomicOr(&bad_val[note][wq >> 1][kg >> 2], v_bad << (8 * (kg & 3)));
                    bad_any[note][1] = 1;
                }
                uint32_t sc[4];
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    sc[e] = (uint32_t) vs[2 * e] | ((uint32_t) vs[2 * e + 1] << 16);
                }
                uint8_t * base = sV + sv * Lay::VB + (kg >> 3) * (D * 128);
#pragma unroll
                for (int h = 0; h < 4; h++) {  // bytes 2h and 2h + 1 of the 8
                    uint32_t r[4][4];          // [pair of keys][low, high of byte 2h, low, high of byte 2h + 1]
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        const uint32_t x = h < 2 ? vw[2 * e].x : vw[2 * e].y, y = h < 2 ? vw[2 * e + 1].x : vw[2 * e + 1].y;
                        unpack4(__byte_perm(x, y, (h & 1) ? 0x7632u : 0x5410u), half2_of(sc[e]), r[e]);
                    }
#pragma unroll
                    for (int q = 0; q < 4; q++) {
                        const int d = (wq >> 1) * 32 + (wq & 1) * 8 + 2 * h + (q >> 1) + 16 * (q & 1);
                        *reinterpret_cast<uint4 *>(base + d * 128 + (((kg & 7) ^ (d & 7)) << 4)) =
                            make_uint4(r[0][q], r[1][q], r[2][q], r[3][q]);
                    }
                }
            }
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) {
                ptx::mbar_arrive(&v_full[sv]);
            }
        }
    } else if (warp == kQtMma) {
        if (lane == 0 && nblk > 0 && tc_wait(q_full, 0, &abort_flag, a.err)) {
            tc_fence_after();
            constexpr uint32_t idesc_s = idesc_kind_f16(128, kQtKeys, true);
            constexpr uint32_t idesc_o = idesc_kind_f16(128, D, true);
            auto issue_s = [&](int i) -> bool {
                const int sk = i % Lay::NK;
                if (!tc_wait(&k_full[sk], (i / Lay::NK) & 1, &abort_flag, a.err)) {
                    return false;
                }
                tc_fence_after();
                const uint32_t st = ptx::smem_u32(sK + sk * Lay::KB);
                const uint32_t tS = tmem + (uint32_t) ((i & 1) * 128);
#pragma unroll
                for (int kk = 0; kk < D / 16; kk++) {
                    umma_ts(tS, tQ + (uint32_t) (kk * 8), smem_desc_sw128(st + (kk >> 2) * 16384 + (kk & 3) * 32), idesc_s, kk > 0);
                }
                umma_commit(&s_full[i & 1]);
                umma_commit(&k_empty[sk]);
                return true;
            };
            bool ok = issue_s(0) && (nblk < 2 || issue_s(1));
            for (int i = 0; ok && i < nblk; i++) {
                if (!tc_wait(&p_full[i & 1], (i >> 1) & 1, &abort_flag, a.err)) {
                    break;
                }
                const int sv = i % Lay::NV;
                if (!tc_wait(&v_full[sv], (i / Lay::NV) & 1, &abort_flag, a.err)) {
                    break;
                }
                tc_fence_after();
                const uint32_t vt = ptx::smem_u32(sV + sv * Lay::VB);
                const uint32_t tP = tmem + (uint32_t) ((i & 1) * 128);
#pragma unroll
                for (int kk = 0; kk < kQtKeys / 16; kk++) {
                    umma_ts(tO, tP + (uint32_t) (kk * 8), smem_desc_sw128(vt + (kk >> 2) * (D * 128) + (kk & 3) * 32), idesc_o,
                            (i > 0 || kk > 0) ? 1u : 0u);
                }
                umma_commit(&pv_done[i & 1]);
                umma_commit(&v_empty[sv]);
                if (i + 1 == nblk) {
                    umma_commit(o_done);
                }
                if (i + 2 < nblk) {
                    ok = issue_s(i + 2);
                }
            }
        }
    } else {
        // ---- softmax: warp w and w + 4 share the TMEM lanes of quarter w % 4 (two threads a row) ----
        constexpr int  HD    = D / 2;  // dimensions of a thread's half of Q and O
        const int      qq    = warp & 3, hf = warp >> 2;
        const int      row   = qq * 32 + lane, r = r0 + row, i_tok = r / a.G;
        const uint32_t lanes = (uint32_t) (qq * 32) << 16;
        const bool     live  = i_tok < n && row0 + i_tok >= 0 && row0 + i_tok < a.n_tok;
        const int      p     = okay && i_tok < n ? len - n + i_tok : -1;
        const int      lo    = a.window > 0 ? max(0, p - a.window + 1) : 0;
        const int64_t  head  = (int64_t) (hk * a.G + r % a.G) * D + hf * HD;
        float          m = -INFINITY, l = 0.0f;
        bool           ok = true;
        uint32_t       nan_blocks = 0;  // of this thread's half
        auto pair_xchg = [&](int phase, float v, float * other) -> bool {
            xchg[((phase & 1) * 2 + hf) * kQtRows + row] = v;
            __syncwarp();
            if (lane == 0) {
                ptx::mbar_arrive(&xbar[qq]);
            }
            if (!__all_sync(0xffffffffu, tc_wait(&xbar[qq], phase & 1, &abort_flag, a.err))) {
                return false;
            }
            *other = xchg[((phase & 1) * 2 + (hf ^ 1)) * kQtRows + row];
            return true;
        };
        float sc = 1.0f;  // of the scores, with log2 e: never 0, so that a masked score stays -inf
        if (nblk > 0) {
            // Q: a power of two takes the row's largest element into [1, 2), the scale's sign goes into it too
            T1         q[HD];
            const T1 * src = reinterpret_cast<const T1 *>(a.q) + (row0 + i_tok) * a.q_stride + head;
            float      mx  = 0.0f, other = 0.0f;
#pragma unroll
            for (int e = 0; e < HD; e += 8) {
                if constexpr (ALIGNED) {
                    *reinterpret_cast<uint4 *>(q + e) = live ? __ldg(reinterpret_cast<const uint4 *>(src + e)) : make_uint4(0, 0, 0, 0);
                } else {
#pragma unroll
                    for (int f = 0; f < 8; f++) {
                        q[e + f] = live ? src[e + f] : io<T>::from_f(0.0f);
                    }
                }
            }
#pragma unroll
            for (int e = 0; e < HD; e++) {
                mx = fmaxf(mx, fabsf(io<T>::to_f(q[e])));
            }
            ok = pair_xchg(0, mx, &other);
            mx = fmaxf(mx, other);
            int ex = (int) (__float_as_uint(mx) >> 23);
            ex     = mx == 0.0f || ex == 255 ? 127 : min(max(ex, 1), 253);
            float down = __uint_as_float((uint32_t) (254 - ex) << 23);
            if (a.scale_log2 == 0.0f) {
                down = 0.0f;
            } else {
                sc   = fmaxf(fabsf(a.scale_log2) * __uint_as_float((uint32_t) ex << 23), 1.2e-38f);
                down = copysignf(down, a.scale_log2);
            }
            uint32_t v[HD / 2];
#pragma unroll
            for (int b = 0; b < HD / 32; b++) {
#pragma unroll
                for (int w = 0; w < 4; w++) {  // unpack4's order of the dimensions of a word
                    const T1 * z = q + 32 * b + 4 * w;
                    v[16 * b + 4 * w]     = u32_of(__floats2half2_rn(io<T>::to_f(z[0]) * down, io<T>::to_f(z[2]) * down));
                    v[16 * b + 4 * w + 1] = u32_of(__floats2half2_rn(io<T>::to_f(z[16]) * down, io<T>::to_f(z[18]) * down));
                    v[16 * b + 4 * w + 2] = u32_of(__floats2half2_rn(io<T>::to_f(z[1]) * down, io<T>::to_f(z[3]) * down));
                    v[16 * b + 4 * w + 3] = u32_of(__floats2half2_rn(io<T>::to_f(z[17]) * down, io<T>::to_f(z[19]) * down));
                }
            }
            if constexpr (D == 128) {
                tmem_st32(tQ + lanes + (uint32_t) (hf * 32), v);
            } else {
                tmem_st16(tQ + lanes + (uint32_t) (hf * 16), v);
                asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) {
                ptx::mbar_arrive(q_full);
            }
        }
        // keys of block i with a bad value scale that this row sees: their dimensions become NaN
        auto look_at_values = [&](int i) {
            if (bad_any[i % kQtRing][1]) {
                const int key0 = (kb_lo + i) * kQtKeys;
                for (int b = 0; b < HD / 32; b++) {
                    for (int c = 0; c < kQtKeys; c++) {
                        if ((bad_val[i % kQtRing][hf * (HD / 32) + b][c >> 5] >> (c & 31)) & 1u) {
                            nan_blocks |= (uint32_t) (key0 + c >= lo && key0 + c <= p) << b;
                        }
                    }
                }
            }
        };
        int  pv_seen0 = 0, pv_seen1 = 0;
        auto wait_pv  = [&](int k) -> bool {
            const int bb = k & 1, ph = k >> 1;
            int &     seen = bb ? pv_seen1 : pv_seen0;
            if (seen > ph) {
                return true;
            }
            if (!__all_sync(0xffffffffu, tc_wait(&pv_done[bb], ph & 1, &abort_flag, a.err))) {
                return false;
            }
            seen = ph + 1;
            tc_fence_after();
            return true;
        };
        for (int i = 0; ok && i < nblk; i++) {
            if (!__all_sync(0xffffffffu, tc_wait(&s_full[i & 1], (i >> 1) & 1, &abort_flag, a.err))) {
                ok = false;
                break;
            }
            tc_fence_after();
            const uint32_t tS = tmem + lanes + (uint32_t) ((i & 1) * 128);
            uint32_t       x[64];
            tmem_ld32(tS + (uint32_t) (hf * 64), x);
            tmem_ld32(tS + (uint32_t) (hf * 64 + 32), x + 32);
            const int key0 = (kb_lo + i) * kQtKeys + hf * 64;
            if (key0 + 63 > p || key0 < lo) {
#pragma unroll
                for (int c = 0; c < 64; c++) {
                    if (key0 + c > p || key0 + c < lo) {
                        x[c] = __float_as_uint(-INFINITY);
                    }
                }
            }
            if (bad_any[i % kQtRing][0]) {
#pragma unroll
                for (int c = 0; c < 64; c++) {
                    if ((bad_key[i % kQtRing][hf * 2 + (c >> 5)] >> (c & 31)) & 1u) {
                        x[c] = __float_as_uint(-INFINITY);
                    }
                }
            }
            float mt[8];
#pragma unroll
            for (int c = 0; c < 8; c++) {
                mt[c] = fmaxf(fmaxf(fmaxf(__uint_as_float(x[c]), __uint_as_float(x[c + 8])),
                                    fmaxf(__uint_as_float(x[c + 16]), __uint_as_float(x[c + 24]))),
                              fmaxf(fmaxf(__uint_as_float(x[c + 32]), __uint_as_float(x[c + 40])),
                                    fmaxf(__uint_as_float(x[c + 48]), __uint_as_float(x[c + 56]))));
            }
            const float mh = fmaxf(fmaxf(fmaxf(mt[0], mt[1]), fmaxf(mt[2], mt[3])), fmaxf(fmaxf(mt[4], mt[5]), fmaxf(mt[6], mt[7])));
            // the exchange also puts both threads' reads of this S buffer before either's P
            float mo;
            if (!pair_xchg(i + 1, mh, &mo)) {
                ok = false;
                break;
            }
            const float mb    = fmaxf(mh, mo) * sc;
            float       alpha = 1.0f;
            bool        resc  = false;
            if (m == -INFINITY) {
                m = mb;
            } else if (mb > m + kQtLag) {
                alpha = ex2_fast(m - mb);
                m     = mb;
                resc  = true;
            }
            const float nm    = m == -INFINITY ? 0.0f : kQtLift - m;
            float       ps[4] = { 0.0f, 0.0f, 0.0f, 0.0f };
            uint32_t    ph[32];
#pragma unroll
            for (int e = 0; e < 32; e++) {
                const float e0 = ex2_fast(fmaf(__uint_as_float(x[2 * e]), sc, nm));
                const float e1 = ex2_fast(fmaf(__uint_as_float(x[2 * e + 1]), sc, nm));
                ps[e & 1] += e0;
                ps[2 + (e & 1)] += e1;
                ph[e] = u32_of(__floats2half2_rn(e0, e1));
            }
            if (i >= 2) {
                if (!wait_pv(i - 2)) {
                    ok = false;
                    break;
                }
                look_at_values(i - 2);
            }
            if (__any_sync(0xffffffffu, resc)) {
                if (!wait_pv(i - 1)) {
                    ok = false;
                    break;
                }
#pragma unroll 1
                for (int c = 0; c < HD / 32; c++) {
                    uint32_t       o[32];
                    const uint32_t col = (uint32_t) (hf * HD + c * 32);
                    tmem_ld32(tO + lanes + col, o);
#pragma unroll
                    for (int e = 0; e < 32; e++) {
                        o[e] = __float_as_uint(__uint_as_float(o[e]) * alpha);
                    }
                    tmem_st32(tO + lanes + col, o);
                }
            }
            l = l * alpha + ((ps[0] + ps[1]) + (ps[2] + ps[3]));
            tmem_st32(tS + (uint32_t) (hf * 32), ph);
            tc_fence_before();
            __syncwarp();
            if (lane == 0) {
                ptx::mbar_arrive(&p_full[i & 1]);
            }
        }
        if (ok && nblk > 0) {
            ok = __all_sync(0xffffffffu, tc_wait(o_done, 0, &abort_flag, a.err));
            tc_fence_after();
            for (int i = max(0, nblk - 2); ok && i < nblk; i++) {
                look_at_values(i);
            }
        }
        float lo_sum = 0.0f;
        if (ok && nblk > 0) {
            ok = pair_xchg(nblk + 1, l, &lo_sum);
        }
        const float lt  = ok ? l + lo_sum : 0.0f;
        const float inv = lt != 0.0f ? 1.0f / lt : 0.0f;
        T1 *        y   = reinterpret_cast<T1 *>(a.o) + (row0 + i_tok) * a.o_stride + head;
#pragma unroll 1
        for (int c = 0; c < HD / 32; c++) {
            uint32_t o[32];
            if (nblk > 0 && ok) {
                tmem_ld32(tO + lanes + (uint32_t) (hf * HD + c * 32), o);
            } else {
#pragma unroll
                for (int e = 0; e < 32; e++) {
                    o[e] = 0u;
                }
            }
            const float f = (nan_blocks >> c) & 1u ? NAN : inv;
            if (live) {
#pragma unroll
                for (int e = 0; e < 32; e += 8) {
                    vec16<T> out;
#pragma unroll
                    for (int g = 0; g < 8; g++) {
                        out.set(g, __uint_as_float(o[e + g]) * f);
                    }
                    if constexpr (ALIGNED) {
                        out.store(y + c * 32 + e);
                    } else {
#pragma unroll
                        for (int g = 0; g < 8; g++) {
                            y[c * 32 + e + g] = out.v[g];
                        }
                    }
                }
            }
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == kQtMma) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512));
    }
}

template <int T, int D> void (*tc_kernel(bool aligned))(const AttnQ4Args) {
    return aligned ? attn_q4_tc_kernel<T, D, true> : attn_q4_tc_kernel<T, D, false>;
}

}  // namespace

// From 64 rows on (half a tile) the tiles of 128 win over tiles of 16 that unpack every key again.
bool attn_q4_tc_wanted(const AttnQ4Args & a, int type, int head_dim) {
    return type != ACB_TYPE_F32 && head_dim <= 128 && (int64_t) a.max_q * a.G >= 64;
}

acb_status attn_q4_tc_launch(const AttnQ4Args & a, int type, int head_dim, cudaStream_t st) {
    const bool aligned = (reinterpret_cast<uintptr_t>(a.q) | reinterpret_cast<uintptr_t>(a.o)) % 16 == 0 && (a.q_stride | a.o_stride) % 8 == 0;
    const auto kern = type == ACB_TYPE_F16 ? (head_dim == 64 ? tc_kernel<ACB_TYPE_F16, 64>(aligned) : tc_kernel<ACB_TYPE_F16, 128>(aligned))
                                           : (head_dim == 64 ? tc_kernel<ACB_TYPE_BF16, 64>(aligned) : tc_kernel<ACB_TYPE_BF16, 128>(aligned));
    const size_t      smem = (size_t) (head_dim == 64 ? QtLayout<64>::TOTAL : QtLayout<128>::TOTAL) + 1024 + 256;
    const cudaError_t e    = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int) smem);
    if (e != cudaSuccess) {
        set_last_cuda_error(e);
        return ACB_ERR_CUDA;
    }
    const int64_t rows = (int64_t) a.max_q * a.G;
    kern<<<dim3((unsigned) ((rows + kQtRows - 1) / kQtRows), (unsigned) a.kv.nkv, (unsigned) a.kv.n_seq), kQtThreads, smem, st>>>(a);
    return launch_status();
}

}  // namespace acb
