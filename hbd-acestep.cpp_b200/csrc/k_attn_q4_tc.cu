// k_attn_q4_tc.cu -- attention over the paged 4-bit KV cache for chunks of prompts, on the 5th-generation tensor cores.
//
// One CTA per 256 rows (new token * G + query head of the group) of a sequence and kv head, in two tiles of 128; key blocks of
// 128. Every cached value is an f16 number, so nothing is rounded on the way into the tiles. 16 warps, the most that leave a
// thread 128 registers:
//   0..3, 4..7  softmax of tile 0 and of tile 1, a thread a row (a TMEM lane): 64 scores of half a block at a time, in registers
//               once for the maximum and the exponentials; P goes back over them as f16 (half a step of 2^-11 of each
//               weight, as k_attn_q4.cu says; their sum is of the unrounded ones);
//   8..11       unpacking V^T: a thread 8 keys by 16 dimensions: the words of two keys are merged by halves, so that unpack4
//               gives pairs of keys, and four pairs make the 16-byte unit of a dimension;
//   12, 13      unpacking K: a thread two keys; the 8 dimensions of a word of codes make one 16-byte unit in the order that
//               unpack4 gives them, and Q is written in the same order (a product does not depend on the order of its k
//               index);
//   14, 15      the products of tile 0 and of tile 1: S = Q K^T of 64 keys from shared memory, O += P V with P from TMEM. The two
//               halves of a block have score columns of their own, so that while the softmax is at one the other's next scores
//               are computed: a softmax never waits for its own product.
// Per key block and tile the tensor cores need 1280 cycles (D = 128; products of 64 columns are bound by shared memory, 48
// cycles where 32 would do) and the exponentials 1024.
//
// 4 sequences with 1200-2048 new rows over 2048-5000 keys (16/8 heads of 128, bf16): 244 us, 726 TFLOP/s. A block takes about
// 4300 cycles, all of which both softmaxes are at work (of a half: wait and load 550, maximum 220, exponentials 1000-1400, signals
// 150). No part bounds it alone: with four unpacking warps (248 us), taking out the exponentials left 243, the products 239,
// three quarters of the unpacking 222, the last and either of the others 200; issue is 52% busy, and the last blocks of the
// grid leave 16% of the SMs idle. Slower were: scores of whole blocks, whose turn waits for the products (303 us); one warp for
// both tiles' products (295, and 393 by a thread behind branches instead of a warp in uniform registers); four warps each
// for K and for V with the registers split by setmaxnreg (254); the next half's scores on their way under the
// exponentials (269); weights taken before the maximum is known and repeated where it moves (260), or with their sum
// in the maximum's place (256); loads of codes along the rows (a quarter of the cache traffic, 250); every sequence's own last
// rows first (251); two threads a row (462), eight warps on one tile (376), the products issued by softmax warps (363).
//
// Every wait is bounded, as in k_attn_tc.cu.
#include <algorithm>

#include "attn_q4.cuh"
#include "ptx.cuh"
#include "tc.cuh"

namespace acb {
namespace {

constexpr int   kQtRows    = 128;  // of a tile
constexpr int   kQtKeys    = 128;  // of a block; scores come 64 keys at a time
constexpr int   kQtHalf    = kQtKeys / 2;
constexpr int   kQtSoft    = 8;   // softmax warps
constexpr int   kQtUnpackV = 4, kQtUnpackK = 2;  // unpacking warps
constexpr int   kQtMma     = kQtSoft + kQtUnpackV + kQtUnpackK;  // and the next: up to 16 warps leave every thread 128 registers
constexpr int   kQtThreads = 32 * (kQtMma + 2);
constexpr float kQtLag     = 8.0f;  // the reference maximum moves when exceeded by more than 2^kQtLag
constexpr float kQtLift    = 6.0f;  // P is held times 2^kQtLift: at most 2^14
constexpr int   kQtRing    = 8;     // blocks whose notes are kept

template <int D> struct QtLayout {
    static constexpr int QB = kQtRows * D * 2, KB = kQtKeys * D * 2, VB = kQtKeys * D * 2, NK = 2, NV = 2;
    static constexpr int TOTAL = 2 * QB + NK * KB + NV * VB;
    // TMEM columns: S/P of a tile's halves of a block at 128 t and 128 t + 64, O at 256 and 384
};

// two f32 in one operation (sm_100)
__device__ __forceinline__ uint64_t pack2(float x, float y) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(x), "f"(y));
    return r;
}

__device__ __forceinline__ void unpack2(uint64_t v, float * x, float * y) {
    asm("mov.b64 {%0, %1}, %2;" : "=f"(*x), "=f"(*y) : "l"(v));
}

__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}

__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}

// 64 columns of this warp's lanes. Load and wait are one statement: nothing can move or copy r in between, and the pairs stay
// where two-element operations want them.
__device__ __forceinline__ void tmem_ld64(uint32_t taddr, uint32_t * r) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x64.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
        "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,"
        "%32,%33,%34,%35,%36,%37,%38,%39,%40,%41,%42,%43,%44,%45,%46,%47,"
        "%48,%49,%50,%51,%52,%53,%54,%55,%56,%57,%58,%59,%60,%61,%62,%63}, [%64];\n\t"
        "tcgen05.wait::ld.sync.aligned;"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
          "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
          "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
          "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31]),
          "=r"(r[32]), "=r"(r[33]), "=r"(r[34]), "=r"(r[35]), "=r"(r[36]), "=r"(r[37]), "=r"(r[38]), "=r"(r[39]),
          "=r"(r[40]), "=r"(r[41]), "=r"(r[42]), "=r"(r[43]), "=r"(r[44]), "=r"(r[45]), "=r"(r[46]), "=r"(r[47]),
          "=r"(r[48]), "=r"(r[49]), "=r"(r[50]), "=r"(r[51]), "=r"(r[52]), "=r"(r[53]), "=r"(r[54]), "=r"(r[55]),
          "=r"(r[56]), "=r"(r[57]), "=r"(r[58]), "=r"(r[59]), "=r"(r[60]), "=r"(r[61]), "=r"(r[62]), "=r"(r[63])
        : "r"(taddr)
        : "memory");
}

// The products' warp runs as one, with everything in uniform registers, and one lane of it issues. A thread alone between
// branches spends more time on moving descriptors and looking at barriers than the tensor cores on the products.
constexpr uint32_t kQtDescHi = (1024u >> 4) | (1u << 14) | (2u << 29);  // smem_desc_sw128's upper word

__device__ __forceinline__ void issue_ss(uint32_t leader, uint32_t d, uint32_t a_lo, uint32_t b_lo, uint32_t idesc, uint32_t acc) {
    asm volatile(
        "{\n\t.reg .pred p, q;\n\t.reg .b64 da, db;\n\tsetp.ne.b32 q, %0, 0;\n\tsetp.ne.b32 p, %5, 0;\n\t"
        "mov.b64 da, {%2, %6};\n\tmov.b64 db, {%3, %6};\n\t"
        "@q tcgen05.mma.cta_group::1.kind::f16 [%1], da, db, %4, p;\n\t}" ::"r"(leader),
        "r"(d), "r"(a_lo), "r"(b_lo), "r"(idesc), "r"(acc), "r"(kQtDescHi));
}

__device__ __forceinline__ void issue_ts(uint32_t leader, uint32_t d, uint32_t a_tmem, uint32_t b_lo, uint32_t idesc, uint32_t acc) {
    asm volatile(
        "{\n\t.reg .pred p, q;\n\t.reg .b64 db;\n\tsetp.ne.b32 q, %0, 0;\n\tsetp.ne.b32 p, %5, 0;\n\t"
        "mov.b64 db, {%3, %6};\n\t"
        "@q tcgen05.mma.cta_group::1.kind::f16 [%1], [%2], db, %4, p;\n\t}" ::"r"(leader),
        "r"(d), "r"(a_tmem), "r"(b_lo), "r"(idesc), "r"(acc), "r"(kQtDescHi));
}

__device__ __forceinline__ void issue_commit(uint32_t leader, uint32_t bar) {
    asm volatile(
        "{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %0, 0;\n\t"
        "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%1];\n\t}" ::"r"(leader),
        "r"(bar)
        : "memory");
}

// of a warp; what is there already costs one look
__device__ __forceinline__ bool warp_wait(uint64_t * bar, uint32_t parity, volatile int * abort_flag, int * err) {
    return __all_sync(0xffffffffu, ptx::mbar_try_wait(bar, parity)) ||
           __all_sync(0xffffffffu, tc_wait(bar, parity, abort_flag, err));
}

template <int T, int D, bool ALIGNED> __global__ void __launch_bounds__(kQtThreads, 1) attn_q4_tc_kernel(const AttnQ4Args a) {
    using Lay = QtLayout<D>;
    using T1  = typename io<T>::t;
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    uint8_t *  sQ      = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint8_t *  sK      = sQ + 2 * Lay::QB;
    uint8_t *  sV      = sK + Lay::NK * Lay::KB;
    uint64_t * q_full  = reinterpret_cast<uint64_t *>(sV + Lay::NV * Lay::VB);
    uint64_t * k_full  = q_full + 1;
    uint64_t * k_empty = k_full + Lay::NK;
    uint64_t * v_full  = k_empty + Lay::NK;
    uint64_t * v_empty = v_full + Lay::NV;
    // [2 t + h], tile t and half h of a block. Phase i of s_full: S(i, h) is there, and P.V(i - 1, h) done
    uint64_t * s_full  = v_empty + Lay::NV;
    uint64_t * p_full  = s_full + 4;
    uint32_t * tmem_slot = reinterpret_cast<uint32_t *>(p_full + 4);
    __shared__ volatile int abort_flag;
    // notes on a block, for what hardly ever happens: keys whose page is not in the pool, and per 32 dimensions the keys whose
    // value scale is no number (their values are left out of the product, where 0 * NaN would reach the rows that do not see
    // them, and make their dimensions NaN in the rows that do)
    __shared__ uint32_t bad_key[kQtRing][4], bad_val[kQtRing][D / 32][4];
    __shared__ int      bad_any[kQtRing][2];

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int hk = blockIdx.x, s = blockIdx.y;
    int64_t    row0;
    int        n, len;
    const bool okay = seq_bounds(a, s, &row0, &n, &len);
    if (!okay && a.err && threadIdx.x == 0) {
        atomicOr(a.err, ACB_DEVERR_LEN_RANGE);
    }
    // the last rows of every sequence first, they see the most keys: what is left for the end is short
    const int r0 = (int) (gridDim.z - 1 - blockIdx.z) * 2 * kQtRows;
    if (r0 >= n * a.G) {
        return;
    }
    const int tiles = r0 + kQtRows < n * a.G ? 2 : 1;
    const int i0 = r0 / a.G, i1 = min(n - 1, (r0 + 2 * kQtRows - 1) / a.G);
    const int p0 = okay ? len - n + i0 : -1, p1 = okay ? len - n + i1 : -1;
    const int key_lo = a.window > 0 ? max(0, p0 - a.window + 1) : 0;
    const int kb_lo  = key_lo / kQtKeys;
    const int nblk   = p1 < 0 ? 0 : p1 / kQtKeys + 1 - kb_lo;

    if (threadIdx.x == 0) {
        abort_flag = 0;
        ptx::mbar_init(q_full, kQtSoft / 2 * tiles);
        for (int i = 0; i < Lay::NK; i++) {
            ptx::mbar_init(&k_full[i], kQtUnpackK);
            ptx::mbar_init(&k_empty[i], tiles);
        }
        for (int i = 0; i < Lay::NV; i++) {
            ptx::mbar_init(&v_full[i], kQtUnpackV);
            ptx::mbar_init(&v_empty[i], tiles);
        }
        for (int i = 0; i < 4; i++) {
            ptx::mbar_init(&s_full[i], 1);
            ptx::mbar_init(&p_full[i], kQtSoft / 2);
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

    if (warp >= kQtSoft && warp < kQtMma) {
        if (warp >= kQtSoft + kQtUnpackV) {
            // ---- unpacking K: a thread two keys ----
            const int tid = threadIdx.x - 32 * (kQtSoft + kQtUnpackV);
            int       kpg[2] = { 0, 0 };
            if (nblk > 0) {
                kpg[0] = a.kv.page_of(s, min(kb_lo * kQtKeys + tid, p1));
                kpg[1] = a.kv.page_of(s, min(kb_lo * kQtKeys + tid + 64, p1));
            }
            for (int i = 0; i < nblk; i++) {
                const int     key0 = (kb_lo + i) * kQtKeys, note = i % kQtRing, next = (i + 2) % kQtRing, sk = i % Lay::NK;
                // from memory before the wait
                const uint4 * kc[2];
                uint4         code[2];
                Words<D / 64> ksw[2];
                bool          bad[2];
#pragma unroll
                for (int e = 0; e < 2; e++) {
                    const int     key  = key0 + tid + 64 * e;
                    const int64_t krow = kpg[e] < 0 ? 0 : a.kv.row(kpg[e], hk, min(key, p1));
                    bad[e]  = kpg[e] < 0;
                    kc[e]   = reinterpret_cast<const uint4 *>(a.kv.kc + krow * (D / 2));
                    code[e] = __ldg(kc[e]);
                    ksw[e].load(a.kv.ks + krow * (D / 32));
                    if (i + 1 < nblk) {
                        kpg[e] = a.kv.page_of(s, min(key + kQtKeys, p1));
                    }
                }
                if (i >= Lay::NK && !warp_wait(&k_empty[sk], (i / Lay::NK - 1) & 1, &abort_flag, a.err)) {
                    break;
                }
                // Room for the notes of block i + 2, where those of block i - 6 are: both tiles' S(i - 2) are done, so both
                // softmaxes are past block i - 3, and no warp is at block i + 2 before this one has filled block i (V of block
                // i + 2 takes the place of block i's, whose products come after).
                if (tid < 4) {
                    bad_key[next][tid] = 0;
                } else if (tid < 6) {
                    bad_any[next][tid - 4] = 0;
                } else if (tid >= 32 && tid < 32 + (D / 32) * 4) {
                    (&bad_val[next][0][0])[tid - 32] = 0;
                }
#pragma unroll
                for (int e = 0; e < 2; e++) {
                    const int  key  = tid + 64 * e;
                    // behind the last row, or before every row's window: no key of this block of rows, wherever its page is
                    const bool gone = key0 + key > p1 || key0 + key < key_lo;
                    if (bad[e] && !gone) {
                        atomicOr(&bad_key[note][key >> 5], 1u << (key & 31));
                        bad_any[note][0] = 1;
                        if (a.err) {
                            atomicOr(a.err, ACB_DEVERR_PAGE_RANGE);
                        }
                    }
                    uint8_t * dst  = sK + sk * Lay::KB + key * 128;
                    uint64_t  sc64 = bad[e] || gone ? 0 : D == 64 ? ksw[e].w[0] : (uint64_t) ksw[e].w[D / 64 - 1] << 32 | ksw[e].w[0];
#pragma unroll 1
                    for (int b = 0; b < D / 32; b++) {  // four words, four 16-byte units
                        const uint4   w4 = code[e];
                        const __half2 sc = __half2half2(__ushort_as_half((uint16_t) sc64));
                        if (b + 1 < D / 32) {
                            code[e] = __ldg(kc[e] + b + 1);
                        }
                        sc64 >>= 16;
                        uint8_t * d = dst + (b >> 1) * 16384;
                        const int u = 4 * (b & 1), x = tid & 7;
                        uint32_t  r[4];
                        unpack4(w4.x, sc, r);
                        *reinterpret_cast<uint4 *>(d + ((u ^ x) << 4)) = make_uint4(r[0], r[1], r[2], r[3]);
                        unpack4(w4.y, sc, r);
                        *reinterpret_cast<uint4 *>(d + (((u + 1) ^ x) << 4)) = make_uint4(r[0], r[1], r[2], r[3]);
                        unpack4(w4.z, sc, r);
                        *reinterpret_cast<uint4 *>(d + (((u + 2) ^ x) << 4)) = make_uint4(r[0], r[1], r[2], r[3]);
                        unpack4(w4.w, sc, r);
                        *reinterpret_cast<uint4 *>(d + (((u + 3) ^ x) << 4)) = make_uint4(r[0], r[1], r[2], r[3]);
                    }
                }
                fence_proxy_async_smem();
                __syncwarp();
                if (lane == 0) {
                    ptx::mbar_arrive(&k_full[sk]);
                }
            }
        } else {
            // ---- unpacking V: a thread 8 keys from 8 kg on (of one page: pages hold 16 or more), 16 dimensions: the 8 bytes from
            // 8 wq on; the lanes of a store phase differ in kg ----
            const int  tid = threadIdx.x & (32 * kQtUnpackV - 1), kg = (tid & 7) | ((tid >> 6) << 3), wq = (tid >> 3) & 7;
            const bool on = D == 128 || wq < 4;  // heads of 64 have 4 such runs
            int        vpg = nblk > 0 ? a.kv.page_of(s, min(kb_lo * kQtKeys + 8 * kg, p1)) : 0;
            for (int i = 0; i < nblk; i++) {
                const int key0 = (kb_lo + i) * kQtKeys, note = i % kQtRing, sv = i % Lay::NV;
                uint2     vw[8];
                uint16_t  vs[8];
                if (on) {
                    const int        j   = key0 + 8 * kg;
                    const int64_t    row = vpg < 0 ? 0 : a.kv.row(vpg, hk, j);
                    const uint8_t *  c   = a.kv.vc + row * (D / 2) + wq * 8;
                    const uint16_t * d   = a.kv.vs + row * (D / 32) + (wq >> 1);
                    const int        in  = vpg < 0 ? 0 : p1 - j + 1;  // keys past the last one: none of their own
#pragma unroll
                    for (int e = 0; e < 8; e++) {
                        vw[e] = e < in ? __ldg(reinterpret_cast<const uint2 *>(c + e * (D / 2))) : make_uint2(0, 0);
                        vs[e] = e < in ? __ldg(d + e * (D / 32)) : (uint16_t) 0;
                    }
                }
                if (i + 1 < nblk) {
                    vpg = a.kv.page_of(s, min(key0 + kQtKeys + 8 * kg, p1));
                }
                if (i >= Lay::NV && !warp_wait(&v_empty[sv], (i / Lay::NV - 1) & 1, &abort_flag, a.err)) {
                    break;
                }
                if (on) {
                    uint32_t sc[4], odd = 0;
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        sc[e] = (uint32_t) vs[2 * e] | ((uint32_t) vs[2 * e + 1] << 16);
                        // exponent field full: adding one unit carries into the sign's place
                        odd |= ((sc[e] & 0x7C007C00u) + 0x04000400u) & 0x80008000u;
                    }
                    if (odd) {
                        uint32_t bits = 0;
#pragma unroll
                        for (int e = 0; e < 8; e++) {
                            if ((vs[e] & 0x7C00u) == 0x7C00u) {
                                sc[e >> 1] &= e & 1 ? 0x0000FFFFu : 0xFFFF0000u;
                                bits |= 1u << e;
                            }
                        }
                        atomicOr(&bad_val[note][wq >> 1][kg >> 2], bits << (8 * (kg & 3)));
                        bad_any[note][1] = 1;
                    }
                    uint8_t * base = sV + sv * Lay::VB + (kg >> 3) * (D * 128);
#pragma unroll 1
                    for (int h = 0; h < 4; h++) {  // bytes 2h and 2h + 1 of the 8
                        uint32_t       r[4][4];    // [pair of keys][low, high of byte 2h, low, high of byte 2h + 1]
                        const uint32_t sel = h & 1 ? 0x7632u : 0x5410u;
#pragma unroll
                        for (int e = 0; e < 4; e++) {
                            const uint32_t x = h < 2 ? vw[2 * e].x : vw[2 * e].y, y = h < 2 ? vw[2 * e + 1].x : vw[2 * e + 1].y;
                            unpack4(__byte_perm(x, y, sel), half2_of(sc[e]), r[e]);
                        }
#pragma unroll
                        for (int q = 0; q < 4; q++) {
                            const int d = (wq >> 1) * 32 + (wq & 1) * 8 + 2 * h + (q >> 1) + 16 * (q & 1);
                            *reinterpret_cast<uint4 *>(base + d * 128 + (((kg & 7) ^ (2 * h + (q >> 1))) << 4)) =
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
        }
    } else if (warp >= kQtMma) {
        // ---- products of tile t ----
        const int      n_blk = __reduce_max_sync(0xffffffffu, warp - kQtMma < tiles ? nblk : 0);
        const int      t     = __reduce_max_sync(0xffffffffu, warp - kQtMma);
        const uint32_t tm    = __reduce_max_sync(0xffffffffu, tmem) + (uint32_t) (t * 128);
        const uint32_t base  = __reduce_max_sync(0xffffffffu, ptx::smem_u32(sQ)) >> 4;  // addresses of descriptors
        const uint32_t bar_s = __reduce_max_sync(0xffffffffu, ptx::smem_u32(s_full + 2 * t));
        const uint32_t leader = lane == 0;
        if (n_blk > 0 && warp_wait(q_full, 0, &abort_flag, a.err)) {
            tc_fence_after();
            constexpr uint32_t idesc_s = idesc_kind_f16(128, kQtHalf, true);
            constexpr uint32_t idesc_o = idesc_kind_f16(128, D, true);
            auto issue_s = [&](int i, int h) {
                const uint32_t q = base + (uint32_t) t * (Lay::QB / 16);
                const uint32_t k = base + (uint32_t) (2 * Lay::QB + (i % Lay::NK) * Lay::KB + h * kQtHalf * 128) / 16;
#pragma unroll
                for (int kk = 0; kk < D / 16; kk++) {
                    const uint32_t off = (uint32_t) ((kk >> 2) * 16384 + (kk & 3) * 32) / 16;
                    issue_ss(leader, tm + (uint32_t) (h * kQtHalf), q + off, k + off, idesc_s, kk > 0);
                }
                issue_commit(leader, bar_s + (uint32_t) h * 8);
            };
            auto issue_pv = [&](int i, int h) {
                const uint32_t v = base + (uint32_t) (2 * Lay::QB + Lay::NK * Lay::KB + (i % Lay::NV) * Lay::VB + h * D * 128) / 16;
#pragma unroll
                for (int kk = 0; kk < kQtHalf / 16; kk++) {
                    issue_ts(leader, tm + 256, tm + (uint32_t) (h * kQtHalf + kk * 8), v + kk * 2, idesc_o,
                             (i > 0 || h > 0 || kk > 0) ? 1u : 0u);
                }
            };
            bool ok = warp_wait(&k_full[0], 0, &abort_flag, a.err);
            if (ok) {
                tc_fence_after();
                issue_s(0, 0);
                issue_s(0, 1);
                issue_commit(leader, ptx::smem_u32(&k_empty[0]));
            }
            for (int i = 0; ok && i < n_blk; i++) {
                const bool more = i + 1 < n_blk;
                ok = warp_wait(&v_full[i % Lay::NV], (i / Lay::NV) & 1, &abort_flag, a.err);
#pragma unroll 1
                for (int h = 0; ok && h < 2; h++) {
                    ok = warp_wait(&p_full[2 * t + h], i & 1, &abort_flag, a.err);
                    if (!ok) {
                        break;
                    }
                    tc_fence_after();
                    issue_pv(i, h);
                    if (!more) {
                        issue_commit(leader, bar_s + (uint32_t) h * 8);
                        continue;
                    }
                    ok = h > 0 || warp_wait(&k_full[(i + 1) % Lay::NK], ((i + 1) / Lay::NK) & 1, &abort_flag, a.err);
                    if (ok) {
                        tc_fence_after();
                        issue_s(i + 1, h);
                    }
                }
                if (ok) {
                    issue_commit(leader, ptx::smem_u32(&v_empty[i % Lay::NV]));
                    if (more) {
                        issue_commit(leader, ptx::smem_u32(&k_empty[(i + 1) % Lay::NK]));
                    }
                }
            }
        }
    } else if ((warp >> 2) < tiles) {
        // ---- softmax: warp w reads TMEM lanes 32 (w % 4).. of tile w / 4 ----
        const int      t = warp >> 2, qq = warp & 3, row = qq * 32 + lane, r = r0 + t * kQtRows + row, i_tok = r / a.G;
        const uint32_t lanes = (uint32_t) (qq * 32) << 16;
        const uint32_t tS = tmem + lanes + (uint32_t) (t * 128), tO = tS + 256;
        const bool     live = i_tok < n && row0 + i_tok >= 0 && row0 + i_tok < a.n_tok;
        const int      p    = okay && i_tok < n ? len - n + i_tok : -1;
        const int      lo   = a.window > 0 ? max(0, p - a.window + 1) : 0;
        const int64_t  head = (int64_t) (hk * a.G + r % a.G) * D;
        float          m = -INFINITY, l = 0.0f;
        float          sc = 1.0f;  // of the scores, with log2 e: never 0, so that a masked score stays -inf
        bool           ok = true;
        uint32_t       nan_blocks = 0;  // 32 dimensions each
        if (nblk > 0) {
            // Q: a power of two takes the row's largest element into [1, 2), the scale's sign goes into it too
            const T1 * src = reinterpret_cast<const T1 *>(a.q) + (row0 + i_tok) * a.q_stride + head;
            float      mx  = 0.0f;
            T1         q[32];  // 32 dimensions at a time, read again once the row's largest is known
            auto       take = [&](int b) {
#pragma unroll
                for (int e = 0; e < 32; e += 8) {
                    if constexpr (ALIGNED) {
                        *reinterpret_cast<uint4 *>(q + e) =
                            live ? __ldg(reinterpret_cast<const uint4 *>(src + 32 * b + e)) : make_uint4(0, 0, 0, 0);
                    } else {
#pragma unroll
                        for (int f = 0; f < 8; f++) {
                            q[e + f] = live ? src[32 * b + e + f] : io<T>::from_f(0.0f);
                        }
                    }
                }
            };
#pragma unroll 1
            for (int b = 0; b < D / 32; b++) {
                take(b);
#pragma unroll
                for (int e = 0; e < 32; e++) {
                    mx = fmaxf(mx, fabsf(io<T>::to_f(q[e])));
                }
            }
            int ex = (int) (__float_as_uint(mx) >> 23);
            ex     = mx == 0.0f || ex == 255 ? 127 : min(max(ex, 1), 253);
            float down = __uint_as_float((uint32_t) (254 - ex) << 23);
            if (a.scale_log2 == 0.0f) {
                down = 0.0f;
            } else {
                sc   = fmaxf(fabsf(a.scale_log2) * __uint_as_float((uint32_t) ex << 23), 1.2e-38f);
                down = copysignf(down, a.scale_log2);
            }
            uint8_t * dst = sQ + t * Lay::QB + row * 128;
#pragma unroll 1
            for (int b = 0; b < D / 32; b++) {
                take(b);
#pragma unroll
                for (int v = 0; v < 4; v++) {  // unit u: the dimensions of word u of the codes in unpack4's order
                    const int      u = 4 * b + v;
                    const T1 *     z = q + 4 * v;
                    const uint32_t w0 = u32_of(__floats2half2_rn(io<T>::to_f(z[0]) * down, io<T>::to_f(z[2]) * down));
                    const uint32_t w1 = u32_of(__floats2half2_rn(io<T>::to_f(z[16]) * down, io<T>::to_f(z[18]) * down));
                    const uint32_t w2 = u32_of(__floats2half2_rn(io<T>::to_f(z[1]) * down, io<T>::to_f(z[3]) * down));
                    const uint32_t w3 = u32_of(__floats2half2_rn(io<T>::to_f(z[17]) * down, io<T>::to_f(z[19]) * down));
                    *reinterpret_cast<uint4 *>(dst + (u >> 3) * 16384 + (((u & 7) ^ (row & 7)) << 4)) = make_uint4(w0, w1, w2, w3);
                }
            }
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) {
                ptx::mbar_arrive(q_full);
            }
        }
        // keys of block i with a bad value scale that this row sees: their dimensions become NaN
        auto look_at_values = [&](int i) {
            if (bad_any[i % kQtRing][1]) {
                const int key0 = (kb_lo + i) * kQtKeys;
#pragma unroll 1
                for (int e = 0; e < (D / 32) * kQtKeys; e++) {
                    const int b = e / kQtKeys, c = e % kQtKeys;
                    if ((bad_val[i % kQtRing][b][c >> 5] >> (c & 31)) & 1u) {
                        nan_blocks |= (uint32_t) (key0 + c >= lo && key0 + c <= p) << b;
                    }
                }
            }
        };
        for (int j = 0; j < 2 * nblk; j++) {
            const int i = j >> 1, h = j & 1;
            ok = warp_wait(&s_full[2 * t + h], i & 1, &abort_flag, a.err);
            if (!ok) {
                break;
            }
            tc_fence_after();
            const uint32_t tH = tS + (uint32_t) (h * kQtHalf);
            if (h == 0 && i > 0) {
                look_at_values(i - 1);
            }
            const int  key0 = (kb_lo + i) * kQtKeys + h * kQtHalf;
            const bool part = __any_sync(0xffffffffu, key0 + kQtHalf - 1 > p || key0 < lo || bad_any[i % kQtRing][0]);
            uint32_t   x[kQtHalf];
            tmem_ld64(tH, x);
            if (part) {
#pragma unroll
                for (int w = 0; w < 2; w++) {  // bit c of see: key k + c is seen
                    const int k   = key0 + 32 * w;
                    uint32_t  see = p < k ? 0u : p >= k + 31 ? ~0u : (2u << (p - k)) - 1u;
                    see &= lo <= k ? ~0u : lo > k + 31 ? 0u : ~0u << (lo - k);
                    see &= ~bad_key[i % kQtRing][2 * h + w];
#pragma unroll
                    for (int c = 0; c < 32; c++) {
                        x[32 * w + c] = (see >> c) & 1u ? x[32 * w + c] : 0xFF800000u;
                    }
                }
            }
            float g[4] = { -INFINITY, -INFINITY, -INFINITY, -INFINITY };
#pragma unroll
            for (int c = 0; c < kQtHalf; c += 2) {
                g[(c >> 1) & 3] = fmaxf(g[(c >> 1) & 3], fmaxf(__uint_as_float(x[c]), __uint_as_float(x[c + 1])));
            }
            const float mb   = fmaxf(fmaxf(g[0], g[1]), fmaxf(g[2], g[3])) * sc;
            bool        resc = false;
            float       alpha = 1.0f;
            if (m == -INFINITY) {
                m = mb;
            } else if (mb > m + kQtLag) {
                alpha = ex2_fast(m - mb);
                m     = mb;
                resc  = true;
            }
            const float nm    = m == -INFINITY ? 0.0f : kQtLift - m;
            const uint64_t sc2 = pack2(sc, sc), nm2 = pack2(nm, nm);
            uint64_t       ps[2] = { 0, 0 };  // sums of weights, two each
#pragma unroll
            for (int w = 0; w < 2; w++) {
                uint32_t ph[16];
#pragma unroll
                for (int e = 0; e < 16; e++) {
                    float e0, e1;
                    unpack2(fma2(pack2(__uint_as_float(x[32 * w + 2 * e]), __uint_as_float(x[32 * w + 2 * e + 1])), sc2, nm2), &e0, &e1);
                    e0        = ex2_fast(e0);
                    e1        = ex2_fast(e1);
                    ps[e & 1] = add2(ps[e & 1], pack2(e0, e1));
                    ph[e]     = u32_of(__floats2half2_rn(e0, e1));
                }
                tmem_st16(tH + (uint32_t) (16 * w), ph);  // over the scores, which are all here
            }
            if (__any_sync(0xffffffffu, resc)) {
                // O is whole once P.V of the half before is done: the other half's next phase (of S of the half after, or of the end)
                ok = j == 0 || warp_wait(&s_full[2 * t + (h ^ 1)], ((j + 1) >> 1) & 1, &abort_flag, a.err);
                if (!ok) {
                    asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
                    break;
                }
                tc_fence_after();
#pragma unroll 1
                for (int c = 0; c < D / 32; c++) {
                    uint32_t o[32];
                    tmem_ld32(tO + (uint32_t) (c * 32), o);
#pragma unroll
                    for (int e = 0; e < 32; e++) {
                        o[e] = __float_as_uint(__uint_as_float(o[e]) * alpha);
                    }
                    tmem_st32(tO + (uint32_t) (c * 32), o);
                }
            }
            float s0, s1, s2, s3;
            unpack2(ps[0], &s0, &s1);
            unpack2(ps[1], &s2, &s3);
            l = l * alpha + ((s0 + s1) + (s2 + s3));
            asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
            tc_fence_before();
            __syncwarp();
            if (lane == 0) {
                ptx::mbar_arrive(&p_full[2 * t + h]);
            }
        }
        if (ok && nblk > 0) {
            ok = warp_wait(&s_full[2 * t], nblk & 1, &abort_flag, a.err) && warp_wait(&s_full[2 * t + 1], nblk & 1, &abort_flag, a.err);
            tc_fence_after();
            if (ok) {
                look_at_values(nblk - 1);
            }
        }
        const float inv = ok && l != 0.0f ? 1.0f / l : 0.0f;
        T1 *        y   = reinterpret_cast<T1 *>(a.o) + (row0 + i_tok) * a.o_stride + head;
#pragma unroll 1
        for (int c = 0; c < D / 32; c++) {
            uint32_t o[32];
            if (nblk > 0 && ok) {
                tmem_ld32(tO + (uint32_t) (c * 32), o);
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

// Which form: here a block goes through all keys of up to 256 rows, 2.0 us for 128 keys, in as many waves as the blocks need; the
// other form cuts the keys over the whole GPU, 70 ps for a key and tile of 16 rows (D = 128). So this one is faster from
// some 180 such tiles of all sequences and kv heads for each wave on. Measured, here and there: 24 sequences of 3000 keys, 8 kv
// heads, 16 rows each 115 us and 93, 32 rows 115 and 162; 4 of 4000, 64 rows 70 and 61, 128 rows 70 and 148; one of 20000,
// 64 rows 314 and 65, 256 rows 360 and 200; 24 of 3000, 2 kv heads of 64, 48 rows 49 and 32, 64 rows 49 and 53. The rows are
// taken as the sequences' mean. With few keys, or where the other form has no workspace to cut them, 64 rows are the border.
bool attn_q4_tc_wanted(const AttnQ4Args & a, int type, int head_dim) {
    const int64_t rows = (int64_t) a.max_q * a.G;
    if (type == ACB_TYPE_F32 || head_dim > 128 || rows > 65535 * 2 * kQtRows) {
        return false;
    }
    const int64_t keys = a.window > 0 ? std::min<int64_t>(a.max_kv, (int64_t) a.window + a.max_q) : a.max_kv;
    if (rows >= 64 && (keys < 512 || a.n_split == 1)) {
        return true;
    }
    const int64_t mean  = (a.rows * a.G + a.kv.n_seq - 1) / a.kv.n_seq, tasks = (int64_t) a.kv.n_seq * a.kv.nkv;
    const int64_t waves = (tasks * ((mean + 2 * kQtRows - 1) / (2 * kQtRows)) + num_sms() - 1) / num_sms();
    return keys >= 512 && tasks * ((mean + 15) / 16) >= 180 * waves;
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
    kern<<<dim3((unsigned) a.kv.nkv, (unsigned) a.kv.n_seq, (unsigned) ((rows + 2 * kQtRows - 1) / (2 * kQtRows))), kQtThreads, smem, st>>>(a);
    return launch_status();
}

}  // namespace acb
