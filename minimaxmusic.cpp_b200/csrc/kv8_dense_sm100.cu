// kv8_dense_sm100.cu - attention over the 8-bit paged KV cache for many query rows (prefill, chunks of a
// prompt) on the 5th-generation tensor cores (tcgen05 + TMEM), sm_100a.
//
// Rows of a unit (kv head, sequence) are (query, head of the group) pairs in that order, so that all query heads of
// a kv head share each K/V tile.  Q is brought to [2^14, 2^15) at its row's largest element by a power of two and
// rounded to F16 (what a 16-bit q has is kept, but for elements below 2^-28 of the largest); an F32 result takes its F16 remainder as a second operand (QP = 2), an F32 or F16 result that of
// the weights P (PP = 2): the product then runs twice, the remainder first, where the accumulator is small.
//
// The tensor core truncates what it adds to an F32 accumulator: each of a tile's K = 16 steps loses up to 2^-23 of
// it, always towards zero.  Over thousands of keys that is 1e-5 and more (measured 7e-7 a tile of 128 keys), so
// two forms:
//   TWO       256 rows per CTA, two 128-row tiles t, O_t accumulated in TMEM over all tiles: BF16 results,
//             whose half step is 2e-3, over up to KE_LONG tokens.
//   not TWO   128 rows per CTA; each tile's P V starts afresh in one of two TMEM buffers, and a warpgroup adds it
//             to O in registers, rounded to nearest.
// 512 threads:
//   warpgroup 0   converts: codes of a 128-key tile go from global memory through registers (loaded one tile
//                 ahead) into F16, which holds them exactly, in 128-byte-swizzled shared memory; the
//                 scales of the tile's pages beside them.
//   warpgroup 1   its first warp allocates TMEM and issues every tcgen05.mma, P being in TMEM over S.
//                 TWO: S_t in columns [128 t, ..), O_t in [256 + D t, ..), in the order QK0(j), PV1(j-1), QK1(j),
//                 PV0(j): one tile's softmax runs beside the other's products.  Otherwise S and P V of tile j in
//                 buffers j & 1, in the order QK(j+1), PV(j): the products of one tile beside the softmax of the next.
//   warpgroup 2   softmax, one row per thread.   warpgroup 3   the same for tile 1 (TWO), or O's sums.
//
// Where the blocks of rows are fewer than half the SMs, each block's key tiles are cut into parts, one CTA each, all at
// once; a part leaves O, m, l and R in the workspace, and the last to arrive joins them in their order.  256 tokens
// over 8192 (one sequence, 32 heads on 8, D = 128, BF16): 65 us against 190 in one part each.
//
// Softmax.  s = S * (row factor * key scale of the column's page), in log2 units; weights 2^(s - m); the
// value scale b = f 2^e of a page is multiplied into them, P = 2^(s - m) * 2^(m + e - R + KE_OFF) * f, so
// that O is in units of 2^(R - KE_OFF).  m and R (the largest s + e of any page) are lazy: a tile's weights are
// taken with those of the tiles before, in one pass, and again with its own only by the rows where the weights of
// a group of 16 columns, times f, sum to more than 2^15 (F16 holds 2^16) or the sum leaves F32's range; O is multiplied
// then.  Finding the maxima first, in a pass of their own: 396 us for the 2048 rows below, 331 so.
//
// Bound: for BF16 the exponentials (16 a cycle and SM: 2048 cycles for 256 rows of a tile, of which the polynomial
// takes 1 in 8: 331 us against 399 without it for 2048 rows over 8192 keys, 32 heads), as many cycles of products
// at D = 128, and the issue of the conversions (about 470 slots a scheduler), which overlap in part: a tile
// pair takes 5100 cycles.  For F32 the products (2048 cycles for 128 rows of a tile) beside a softmax of 3000.
#include "kv8.cuh"
#include "tc_sm100.cuh"

#include <algorithm>

namespace mm3fa {

constexpr int KE_THREADS = 512;
constexpr int KE_M       = 128;  // rows per Q tile
constexpr int KE_N       = 128;  // keys per tile
constexpr int KE_TMEM    = 512;
constexpr int KE_EMU     = 1;    // of every 8 pairs of weights, those by polynomial where P is rounded to F16 anyway
constexpr int KE_OFF     = 8;    // P is held times 2^8 at the maxima: a tile's may be 2^7 above those taken before
// Tiles of a part, at least: 1, 2, 4 take 25.2, 24.4, 28.4 us for 64 tokens over 1000 (BF16), 32.6, 28.3, 30.3 over 2000.
constexpr int KE_PART  = 2;
constexpr int KE_PARTS = 32;  // parts of a block of rows, at most: a joining thread holds a factor of each
constexpr int KE_REGS_LAUNCH  = 128;  // 65536 / 512
constexpr int KE_REGS_SOFTMAX = 192;  // 2 x 192 + 96 + 32 = 4 x 128
constexpr int KE_REGS_CONVERT = 96;
constexpr int KE_REGS_ISSUE   = 32;
static_assert(2 * KE_REGS_SOFTMAX + KE_REGS_CONVERT + KE_REGS_ISSUE <= 4 * KE_REGS_LAUNCH, "more registers than the launch has");

// Tokens up to which the truncated sums in TMEM (7e-7 of the result a tile of 128) stay a fifth of BF16's half step.
constexpr int KE_LONG = 65536;

template <int D, int QP, bool TWO>
struct KeSmem {
    static constexpr int HALVES = D / 64;             // 128-byte column blocks
    static constexpr int QT     = HALVES * KE_M * 128;
    static constexpr int KT     = HALVES * KE_N * 128;
    static constexpr int NK = 2, NV = 2;
    static constexpr int OFF_Q    = 0;                                  // [tile][part]
    static constexpr int OFF_K    = OFF_Q + (TWO ? 2 : 1) * QP * QT;    // [NK]
    static constexpr int OFF_V    = OFF_K + NK * KT;                    // [NV]
    static constexpr int OFF_SC   = OFF_V + NV * KT;                    // [4 tiles][8 groups] (a, f, e, present)
    static constexpr int OFF_G    = OFF_SC + 4 * 8 * 16;                // [4 tiles][row] growth of R, then [2][row]
    static constexpr int OFF_F    = OFF_G + (TWO ? 0 : 6 * KE_M * 4);   // [tile][row] factors of the rows
    static constexpr int OFF_BAR  = OFF_F + (TWO ? 2 : 1) * KE_M * 4;
    static constexpr int OFF_MISC = OFF_BAR + 32 * 8;
    static constexpr int TOTAL    = OFF_MISC + 32 + 1024;               // + alignment
};

enum : int {
    KB_KFULL  = 0,   // [2] 128 converting threads
    KB_KEMPTY = 2,   // [2]
    KB_VFULL  = 4,   // [2]
    KB_VEMPTY = 6,   // [2]
    KB_SFULL  = 8,   // [2] per Q tile (TWO) or S buffer
    KB_PREADY = 10,  // [2] 128 softmax threads
    KB_OFULL  = 12,  // [2] the last P V of a Q tile (TWO), or the P V of a tile in a buffer
    KB_QREADY = 14,  // [2] 256: those that stage a Q tile, 128 threads twice (TWO) or the 256 of warpgroups 2 and 3
    KB_SCALES = 16,  // [4] 8 converting threads: a ring deeper than K's, for a softmax that is behind the products
    KB_GROW   = 20,  // [4] 128 softmax threads (not TWO): the growth of a tile's R, read beside its P V
    KB_OFREE  = 24,  // [2] 128 summing threads (not TWO)
    KB_LAST   = 26,  // 128 softmax threads (not TWO): the rows' sums
    KB_DONE   = 27,
    KB_COUNT  = 28,
};

__host__ __device__ constexpr uint32_t ke_arrivals(int b) {
    return b == KB_QREADY || b == KB_QREADY + 1 ? 256u :
           b < KB_KEMPTY || (b >= KB_VFULL && b < KB_VEMPTY) || (b >= KB_PREADY && b < KB_OFULL) || (b >= KB_QREADY && b < KB_SCALES) ||
                   (b >= KB_GROW && b < KB_DONE)
               ? 128u
               : (b >= KB_SCALES && b < KB_GROW ? 8u : 1u);
}

__device__ __forceinline__ uint64_t fmul2(uint64_t a, uint64_t b) {
    uint64_t d;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}

__device__ __forceinline__ uint32_t ke_pack(float lo, float hi) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t *>(&h);
}

// 16 codes -> 16 F16 numbers (0x6400 | u is 1024 + u; less 1152 the code)
__device__ __forceinline__ void ke_convert(const uint4 & c, uint4 & lo, uint4 & hi) {
    const uint32_t bias = 0x64806480u;
    uint32_t       w[8];
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const uint32_t u = (&c.x)[i] ^ 0x80808080u;
#pragma unroll
        for (int k = 0; k < 2; k++) {
            const uint32_t x = __byte_perm(u, 0x64646464u, k ? 0x4342 : 0x4140);
            const __half2  h = __hsub2(*reinterpret_cast<const __half2 *>(&x), *reinterpret_cast<const __half2 *>(&bias));
            w[2 * i + k]     = *reinterpret_cast<const uint32_t *>(&h);
        }
    }
    lo = make_uint4(w[0], w[1], w[2], w[3]);
    hi = make_uint4(w[4], w[5], w[6], w[7]);
}

// kind::f16 instruction descriptor: F16 x F16 -> F32, M = 128
__host__ __device__ constexpr uint32_t ke_idesc(int n, bool b_mn_major) {
    return (1u << 4) | ((b_mn_major ? 1u : 0u) << 16) | ((uint32_t) (n >> 3) << 17) | ((uint32_t) (KE_M >> 4) << 24);
}

template <int D, int QP, int PP, bool TWO, bool CAP>
__global__ void __launch_bounds__(KE_THREADS, 1) kv8_dense_kernel(const Kv8AttnParams p) {
    using L          = KeSmem<D, QP, TWO>;
    constexpr int NK = L::NK, NV = L::NV, KE_ROWS = TWO ? 256 : 128;
    constexpr int ESZ = QP == 2 ? 4 : 2;  // bytes of a result value: F32 where Q has two parts
    extern __shared__ __align__(16) char smem_raw[];
    char *     smem      = smem_raw + ((1024u - (smem_addr(smem_raw) & 1023u)) & 1023u);
    uint64_t * bar       = reinterpret_cast<uint64_t *>(smem + L::OFF_BAR);
    uint32_t * tmem_slot = reinterpret_cast<uint32_t *>(smem + L::OFF_MISC);
    int *      abort_f   = reinterpret_cast<int *>(smem + L::OFF_MISC + 4);
    float4 *   scales    = reinterpret_cast<float4 *>(smem + L::OFF_SC);
    float *    grows     = reinterpret_cast<float *>(smem + L::OFF_G);
    float *    factors   = reinterpret_cast<float *>(smem + L::OFF_F);

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, wg = warp >> 2;
    if (tid == 0) {
        for (int i = 0; i < KB_COUNT; i++) {
            mbar_init(&bar[i], ke_arrivals(i));
        }
        *abort_f = 0;
        fence_mbar_init();
    }
    if (warp == 4) {
        tmem_alloc(tmem_slot, KE_TMEM);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    kv8_dep_wait();
    const uint64_t deadline = global_timer_ns() + p.timeout_ns;  // the time of the kernel before is not this one's

    // ---- the work item: row blocks last first, so that the longest causal ones start first
    const int hs = p.c.n_head_kv * p.t.n_seq, all_rows = p.ratio * p.n_q;
    const int items = (int) gridDim.x / p.parts, item = (int) blockIdx.x % items, part = (int) blockIdx.x / items;
    const int blk = (all_rows + KE_ROWS - 1) / KE_ROWS - 1 - item / hs;
    const int h = item % hs % p.c.n_head_kv, s = item % hs / p.c.n_head_kv;
    const int nq = p.q_len ? min(max(p.q_len[s], 0), p.n_q) : p.n_q;
    const int n  = min(max(p.kv_len[s], 0), p.t.max_pages * p.c.P);
    const int row0 = blk * KE_ROWS, its_rows = min(nq * p.ratio - row0, KE_ROWS);  // rows of this block
    // keys that its last row sees
    const int q_last    = its_rows > 0 ? (row0 + its_rows - 1) / p.ratio : 0;
    const int its_keys  = its_rows > 0 ? (p.causal ? max(n - (nq - 1 - q_last), 0) : n) : 0;
    const int its_tiles = (its_keys + KE_N - 1) / KE_N;
    // this CTA's part of the tiles; a block with few of them has fewer parts
    const int  parts = min(p.parts, max(1, (its_tiles + KE_PART - 1) / KE_PART));
    const int  tile0 = (int) ((unsigned) its_tiles * (unsigned) min(part, parts) / (unsigned) parts);
    const int  tiles = (int) ((unsigned) its_tiles * (unsigned) min(part + 1, parts) / (unsigned) parts) - tile0;
    const int  rows  = part < parts ? its_rows : 0, before = tile0 * KE_N, keys = its_keys - before;
    const bool two   = TWO && rows > KE_M;

    if (wg == 0) {
        // ======================================================= conversion
        regs_dec<KE_REGS_CONVERT>();
        constexpr int LD = D / 16 * KE_N / 128;  // 16-code pieces per thread and tile
        // thread: rows 32 warp + 8 i + (lane & 7), pieces (lane >> 3) + 4 k: a warp reads whole 64-byte runs, and the
        // stores of eight lanes fall into eight rows, so into different banks
        const int * row = p.t.pages + (int64_t) s * p.t.stride + (before >> p.c.log2p);
        int         pg0 = -1, pg1 = -1;
        auto        fetch = [&](int j) {  // table entries of the warp's 32 rows of tile j
            const int k0 = j * KE_N + 32 * warp, i = k0 >> p.c.log2p;
            pg0 = k0 < keys ? row[i] : -1;
            pg1 = p.c.log2p == 4 ? (k0 + 16 < keys ? row[i + 1] : -1) : pg0;
        };
        uint4 kx[LD], vx[LD];
        // this lane's place in a 32-row run of codes, and in the F16 tile: piece pc holds the 16-byte chunks 2 pc, 2 pc + 1
        const int      src_off = (lane & 7) * D + (lane >> 3) * 16;
        const uint32_t dst_off = (uint32_t) ((32 * warp + (lane & 7)) * 128 + (((2 * (lane >> 3)) ^ (lane & 7)) << 4));
        auto           load    = [&](int j, const int8_t * pool, uint4 (&x)[LD]) {
            const bool     ok0 = (unsigned) pg0 < (unsigned) p.c.n_pages, ok1 = (unsigned) pg1 < (unsigned) p.c.n_pages;
            const int      in  = (j * KE_N + 32 * warp) & (p.c.P - 1);  // first row of the run in its page
            const int8_t * a   = pool + (((int64_t) (ok0 ? pg0 : 0) * p.c.n_head_kv + h) * p.c.P + in) * D + src_off;
            const int8_t * b   = p.c.log2p > 4 ? a : pool + (((int64_t) (ok1 ? pg1 : 0) * p.c.n_head_kv + h) * p.c.P - 16) * D + src_off;
#pragma unroll
            for (int i = 0; i < LD; i++) {
                const int8_t * at = ((i & 3) < 2 ? a : b) + 8 * (i & 3) * D + 64 * (i >> 2);
                x[i] = make_uint4(0, 0, 0, 0);
                if ((i & 3) < 2 ? ok0 : ok1) {
                    x[i] = __ldg(reinterpret_cast<const uint4 *>(at));
                }
            }
        };
        auto store = [&](char * tile, const uint4 (&x)[LD]) {
            char * to = tile + dst_off, *to1 = tile + (dst_off ^ 16u);
#pragma unroll
            for (int i = 0; i < LD; i++) {
                uint4 a, b;
                ke_convert(x[i], a, b);
                *reinterpret_cast<uint4 *>(to + 8 * (i & 3) * 128 + (i >> 2) * (KE_N * 128))  = a;
                *reinterpret_cast<uint4 *>(to1 + 8 * (i & 3) * 128 + (i >> 2) * (KE_N * 128)) = b;
            }
        };
        bool ok = true;
        if (tiles > 0) {
            fetch(0);
            load(0, p.c.k, kx);
            load(0, p.c.v, vx);
        }
        for (int j = 0; j < tiles; j++) {
            const int sk = j % NK, sv = j % NV;
            if (j + 1 < tiles) {
                fetch(j + 1);
            }
            float4 sc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            if (tid < 8) {  // 16-key groups of the tile
                const int k0 = j * KE_N + 16 * tid, pg = k0 < keys ? row[k0 >> p.c.log2p] : -1;
                if ((unsigned) pg < (unsigned) p.c.n_pages) {
                    const int64_t ph = (int64_t) pg * p.c.n_head_kv + h;
                    const float   v  = p.c.v_scale[ph];
                    const int     e  = min(max((int) (__float_as_uint(v) >> 23 & 255u) - 127, -126), 126);
                    sc = make_float4(p.c.k_scale[ph], v * __uint_as_float((uint32_t) (127 - e) << 23), (float) e, 1.0f);
                }
            }
            if (j >= NK && !mbar_wait_bounded(&bar[KB_KEMPTY + sk], (uint32_t) ((j / NK - 1) & 1), deadline)) {
                ok = false;
                break;
            }
            if (tid < 8) {
                scales[(j & 3) * 8 + tid] = sc;
                dn_mbar_arrive(&bar[KB_SCALES + (j & 3)]);
            }
            store(smem + L::OFF_K + sk * L::KT, kx);
            fence_proxy_async_smem();
            dn_mbar_arrive(&bar[KB_KFULL + sk]);
            if (j + 1 < tiles) {
                load(j + 1, p.c.k, kx);
            }
            if (j >= NV && !mbar_wait_bounded(&bar[KB_VEMPTY + sv], (uint32_t) ((j / NV - 1) & 1), deadline)) {
                ok = false;
                break;
            }
            store(smem + L::OFF_V + sv * L::KT, vx);
            fence_proxy_async_smem();
            dn_mbar_arrive(&bar[KB_VFULL + sv]);
            if (j + 1 < tiles) {
                load(j + 1, p.c.v, vx);
            }
        }
        if (!ok) {
            atomicExch(abort_f, 1);
        }
    } else if (wg == 1) {
        // ======================================================= MMA issue (one warp, elected lane)
        regs_dec<KE_REGS_ISSUE>();
        if (warp == 4) {
            const uint32_t id_qk = ke_idesc(KE_N, false), id_pv = ke_idesc(D, true);
            // descriptors of the buffers' first bytes; an offset adds to the address field (16-byte units)
            const uint64_t q_d = sw128_desc(smem_addr(smem + L::OFF_Q), 16, 1024), k_d = sw128_desc(smem_addr(smem + L::OFF_K), 16, 1024);
            const uint64_t v_d = sw128_desc(smem_addr(smem + L::OFF_V), (uint32_t) (KE_N * 128), 1024);
            // S of tile j of Q tile t (buffer j & 1 where there is one Q tile); the remainder of Q first
            auto qk = [&](int t, int j) {
                const int buf = TWO ? t : j & 1;
                // rolled loops: unrolled ones keep every descriptor in registers that this warpgroup does not have
#pragma unroll 1
                for (int part = QP - 1; part >= 0; part--) {
                    uint64_t a = q_d + (uint64_t) (((t * QP + part) * L::QT) >> 4), b = k_d + (uint64_t) (((j % NK) * L::KT) >> 4);
#pragma unroll 1
                    for (int c = 0; c < L::HALVES; c++) {
#pragma unroll
                        for (int k = 0; k < 4; k++) {
                            umma_f16(tmem + (uint32_t) (buf * KE_N), a + (uint64_t) (2 * k), b + (uint64_t) (2 * k), id_qk, QP - 1 - part + c + k > 0 ? 1u : 0u);
                        }
                        a += (KE_M * 128) >> 4, b += (KE_N * 128) >> 4;
                    }
                }
                umma_commit(&bar[KB_SFULL + buf]);
            };
            auto pv = [&](int t, int j) {
                const int buf = TWO ? t : j & 1;
#pragma unroll 1
                for (int part = PP - 1; part >= 0; part--) {
                    uint32_t a = tmem + (uint32_t) (buf * KE_N + part * 64);
                    uint64_t b = v_d + (uint64_t) (((j % NV) * L::KT) >> 4);
#pragma unroll 1
                    for (int c = 0; c < 2; c++) {
#pragma unroll
                        for (int k = 0; k < 4; k++) {
                            umma_f16_ts(tmem + 256u + (uint32_t) (buf * D), a + (uint32_t) (8 * k), b + (uint64_t) ((k * 16 * 128) >> 4), id_pv,
                                        (TWO ? j : 0) + PP - 1 - part + c + k > 0 ? 1u : 0u);
                        }
                        a += 32, b += (4 * 16 * 128) >> 4;
                    }
                }
            };
            auto wait = [&](int b, int i) {
                const bool ok = dn_wait_warp(&bar[b], (uint32_t) (i & 1), deadline);
                tc_fence_after();
                return ok;
            };
            bool ok = true;
            if (TWO && tiles > 0) {
                ok = wait(KB_QREADY, 0) && wait(KB_KFULL, 0);
                if (ok) {
                    qk(0, 0);
                    if (two) {
                        ok = wait(KB_QREADY + 1, 0);
                        if (ok) {
                            qk(1, 0);
                        }
                    }
                    umma_commit(&bar[KB_KEMPTY]);
                }
                for (int j = 0; ok && j < tiles; j++) {
                    const bool next = j + 1 < tiles;
                    ok = wait(KB_VFULL + j % NV, j / NV) && wait(KB_PREADY, j);
                    if (!ok) {
                        break;
                    }
                    pv(0, j);
                    if (next) {
                        ok = wait(KB_KFULL + (j + 1) % NK, (j + 1) / NK);
                        if (!ok) {
                            break;
                        }
                        qk(0, j + 1);
                    } else {
                        umma_commit(&bar[KB_OFULL]);
                    }
                    if (two) {
                        ok = wait(KB_PREADY + 1, j);
                        if (!ok) {
                            break;
                        }
                        pv(1, j);
                        umma_commit(&bar[KB_VEMPTY + j % NV]);
                        if (next) {
                            qk(1, j + 1);
                        } else {
                            umma_commit(&bar[KB_OFULL + 1]);
                        }
                    } else {
                        umma_commit(&bar[KB_VEMPTY + j % NV]);
                    }
                    if (next) {
                        umma_commit(&bar[KB_KEMPTY + (j + 1) % NK]);
                    }
                }
            }
            if (!TWO && tiles > 0) {
                ok = wait(KB_QREADY, 0) && wait(KB_KFULL, 0);
                if (ok) {
                    qk(0, 0);
                    umma_commit(&bar[KB_KEMPTY]);
                }
                for (int j = 0; ok && j < tiles; j++) {
                    if (j + 1 < tiles) {  // over P(j - 1), whose product was issued before
                        ok = wait(KB_KFULL + (j + 1) % NK, (j + 1) / NK);
                        if (!ok) {
                            break;
                        }
                        qk(0, j + 1);
                        umma_commit(&bar[KB_KEMPTY + (j + 1) % NK]);
                    }
                    ok = wait(KB_VFULL + j % NV, j / NV) && wait(KB_PREADY + (j & 1), j >> 1) && (j < 2 || wait(KB_OFREE + (j & 1), (j >> 1) - 1));
                    if (!ok) {
                        break;
                    }
                    pv(0, j);
                    umma_commit(&bar[KB_VEMPTY + j % NV]);
                    umma_commit(&bar[KB_OFULL + (j & 1)]);
                }
            }
            if (!ok) {
                atomicExch(abort_f, 1);
            }
            // every MMA issued has to be complete before TMEM and shared memory are given up
            umma_commit(&bar[KB_DONE]);
            dn_wait_warp(&bar[KB_DONE], 0, global_timer_ns() + p.timeout_ns);
        }
    } else {
        // ======================================================= softmax
        regs_inc<KE_REGS_SOFTMAX>();
        const int      t = TWO ? wg - 2 : 0, quad = warp & 3, r = quad * 32 + lane;  // Q tile, TMEM lane quadrant, row of the tile
        const uint32_t tl    = (uint32_t) (quad * 32) << 16;
        const uint32_t o_col = tmem + tl + 256u + (uint32_t) (t * D);
        const int      tile_rows = min(rows - t * KE_M, KE_M);  // may be 0 or less
        char *         qs = smem + L::OFF_Q + t * QP * L::QT;
        // a warp's 32 rows of the result, from the tile's Q, [32 rows][D] with the 16-byte chunks swizzled by the row
        // against bank conflicts: store_rows writes them one after another, each as one run of bytes
        char * mine = qs + quad * 32 * (D * ESZ);
        auto   stage_cols = [&](int c, const uint32_t (&o)[32]) {  // columns 32 c .. of this thread's row
            constexpr int PER = 16 / ESZ;
#pragma unroll
            for (int k = 0; k < 32 / PER; k++) {
                uint4 w;
                if (ESZ == 4) {
                    w = make_uint4(o[4 * k & 31], o[(4 * k + 1) & 31], o[(4 * k + 2) & 31], o[(4 * k + 3) & 31]);
                } else {
                    uint32_t u[4];
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        const float x = __uint_as_float(o[(8 * k + 2 * i) & 31]), y = __uint_as_float(o[(8 * k + 2 * i + 1) & 31]);
                        if (p.o.type == KV_F16) {
                            u[i] = ke_pack(x, y);
                        } else {
                            const __nv_bfloat162 b = __floats2bfloat162_rn(x, y);
                            u[i] = *reinterpret_cast<const uint32_t *>(&b);
                        }
                    }
                    w = make_uint4(u[0], u[1], u[2], u[3]);
                }
                const int ck = c * (32 / PER) + k;
                *reinterpret_cast<uint4 *>(mine + lane * (D * ESZ) + ((ck ^ (lane & 7)) << 4)) = w;
            }
        };
        auto store_rows = [&] {
            __syncwarp();
            constexpr int CK = D * ESZ / 16;  // chunks of a row: 8, 16 or 32
            // lane i: the address of row i
            const int      rl = row0 + t * KE_M + quad * 32 + lane, ql = (int) kv8_div((uint32_t) rl, p.ratio_inv), hl = h * p.ratio + rl - ql * p.ratio;
            const uint64_t al = reinterpret_cast<uint64_t>(p.o.data + (int64_t) hl * p.o.nb1 + (int64_t) ql * p.o.nb2 + (int64_t) s * p.o.nb3);
            if (p.o.vec) {
#pragma unroll 8
                for (int it = 0; it < CK; it++) {
                    const int   i = it * (32 / CK) + lane / CK, ck = lane % CK;  // row of the warp, chunk
                    char *      dst = reinterpret_cast<char *>(__shfl_sync(0xffffffffu, al, i)) + ck * 16;
                    const uint4 w   = *reinterpret_cast<const uint4 *>(mine + i * (D * ESZ) + ((ck ^ (i & 7)) << 4));
                    if (quad * 32 + i < tile_rows) {
                        *reinterpret_cast<uint4 *>(dst) = w;
                    }
                }
                return;
            }
#pragma unroll 1
            for (int it = 0; it < CK; it++) {
                const int   i = it * (32 / CK) + lane / CK, ck = lane % CK;
                char *      dst = reinterpret_cast<char *>(__shfl_sync(0xffffffffu, al, i)) + ck * 16;
                const uint4 w   = *reinterpret_cast<const uint4 *>(mine + i * (D * ESZ) + ((ck ^ (i & 7)) << 4));
                if (quad * 32 + i >= tile_rows) {
                    continue;
                }
                if (ESZ == 4) {
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        reinterpret_cast<uint32_t *>(dst)[e] = (&w.x)[e];
                    }
                } else {
#pragma unroll
                    for (int e = 0; e < 8; e++) {
                        reinterpret_cast<uint16_t *>(dst)[e] = (uint16_t) ((&w.x)[e >> 1] >> (16 * (e & 1)));
                    }
                }
            }
        };
        // ---- parts of a block: each leaves its O, maxima and sums, row r of thread r, and the last to arrive joins them in
        // their order
        constexpr int SLOT = KE_M * (D + 4);  // floats: [D / 4][row] of four, then m, l and R of the rows
        float *       slot = p.part + (int64_t) ((item * p.parts + part) * (TWO ? 2 : 1) + t) * SLOT;
        const int     own  = quad * 32 + lane;
        auto          give = [&](int c, const uint32_t (&o)[32]) {
#pragma unroll
            for (int k = 0; k < 8; k++) {
                reinterpret_cast<uint4 *>(slot)[(c * 8 + k) * KE_M + own] = make_uint4(o[4 * k], o[4 * k + 1], o[4 * k + 2], o[4 * k + 3]);
            }
        };
        auto give_state = [&](float m, float l, float R) {
            slot[D * KE_M + own] = m, slot[(D + 1) * KE_M + own] = l, slot[(D + 2) * KE_M + own] = R;
        };
        auto arrive = [&] {  // by the 128 threads of a Q tile; true for the last part
            int * last = reinterpret_cast<int *>(smem + L::OFF_MISC + 8 + 4 * t);
            __threadfence();
            asm volatile("bar.sync %0, 128;" ::"r"(1 + t) : "memory");
            if (own == 0) {
                uint32_t * count = p.counters + item * 2 + t;
                *last            = atomicAdd(count, 1u) == (uint32_t) (parts - 1);
                if (*last) {
                    *count = 0;
                }
                __threadfence();
            }
            asm volatile("bar.sync %0, 128;" ::"r"(1 + t) : "memory");
            return *reinterpret_cast<volatile int *>(last) != 0;
        };
        auto join = [&] {  // the result's rows from the parts, into shared memory; every product is done
            const float * first = p.part + (int64_t) (item * p.parts * (TWO ? 2 : 1) + t) * SLOT;
            constexpr int STEP  = (TWO ? 2 : 1) * SLOT;
            float         m = -INFINITY, R = -INFINITY, l = 0.0f, f[KE_PARTS];
#pragma unroll 4
            for (int k = 0; k < parts; k++) {
                m = fmaxf(m, __ldcg(first + k * STEP + D * KE_M + own)), R = fmaxf(R, __ldcg(first + k * STEP + (D + 2) * KE_M + own));
            }
#pragma unroll 4
            for (int k = 0; k < parts; k++) {  // (a sum of NaN passes through a factor of 0)
                const float mk = __ldcg(first + k * STEP + D * KE_M + own), Rk = __ldcg(first + k * STEP + (D + 2) * KE_M + own);
                l += __ldcg(first + k * STEP + (D + 1) * KE_M + own) * (mk == -INFINITY ? 0.0f : ex2(mk - m));
                f[k] = Rk == -INFINITY ? 0.0f : ex2(Rk - R);
            }
            const float inv = l != 0.0f ? (1.0f / (1 << KE_OFF)) / l : 0.0f, up = R == -INFINITY ? 0.0f : ex2(R - m);
            // 32 columns of a part at a time through this thread's own places in K's and V's shared memory
            constexpr int  NS   = (TWO ? 2 : 4) * L::KT / (KE_M * 128);
            const uint32_t ring = smem_addr(smem + L::OFF_K + t * 2 * L::KT) + (uint32_t) own * 16;
            int            fc = 0, fk = 0, fs = 0, at = 0;
            auto           fetch = [&] {
                if (fc < D / 32) {
                    const float * src = first + fk * STEP + (fc * 8 * KE_M + own) * 4;
#pragma unroll
                    for (int e = 0; e < 8; e++) {
                        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(ring + (uint32_t) ((fs * 8 + e) * KE_M * 16)),
                                     "l"(src + e * KE_M * 4)
                                     : "memory");
                    }
                    fc = fk + 1 == parts ? fc + 1 : fc, fk = fk + 1 == parts ? 0 : fk + 1;
                }
                fs = fs + 1 == NS ? 0 : fs + 1;
                asm volatile("cp.async.commit_group;" ::: "memory");
            };
#pragma unroll 1
            for (int i = 0; i < NS - 1; i++) {
                fetch();
            }
#pragma unroll 1
            for (int c = 0; c < D / 32; c++) {
                float a[32];
#pragma unroll
                for (int e = 0; e < 32; e++) {
                    a[e] = 0.0f;
                }
#pragma unroll 1
                for (int k = 0; k < parts; k++) {
                    fetch();
                    asm volatile("cp.async.wait_group %0;" ::"n"(NS - 1) : "memory");
                    const float g = f[k];
#pragma unroll
                    for (int e = 0; e < 8; e++) {
                        float4 x;
                        asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];"
                                     : "=f"(x.x), "=f"(x.y), "=f"(x.z), "=f"(x.w)
                                     : "r"(ring + (uint32_t) ((at * 8 + e) * KE_M * 16)));
                        a[4 * e] = fmaf(x.x, g, a[4 * e]), a[4 * e + 1] = fmaf(x.y, g, a[4 * e + 1]);
                        a[4 * e + 2] = fmaf(x.z, g, a[4 * e + 2]), a[4 * e + 3] = fmaf(x.w, g, a[4 * e + 3]);
                    }
                    at = at + 1 == NS ? 0 : at + 1;
                }
                uint32_t o[32];
#pragma unroll
                for (int e = 0; e < 32; e++) {
                    o[e] = __float_as_uint(a[e] * inv * up);
                }
                stage_cols(c, o);
            }
        };
        // ---- Q: rows [ra, ra + 16) of the tile by one warp, whole rows at a time, all loads in flight
        auto stage_q = [&](int ra) {
            constexpr int E = D / 32, B = 8;
            // lane i: the address of row i
            const int      rl = row0 + t * KE_M + ra + (lane & 15), ql = (int) kv8_div((uint32_t) rl, p.ratio_inv), hl = h * p.ratio + rl - ql * p.ratio;
            const uint64_t al = reinterpret_cast<uint64_t>(p.q.data + (int64_t) ql * p.q.nb1 + (int64_t) hl * p.q.nb2 + (int64_t) s * p.q.nb3);
            const int      e0 = lane * E, sub = (e0 % 8) * 2;
            char *         to = qs + (e0 / 64) * (KE_M * 128) + sub;
            const bool     f32 = p.q.type == KV_F32, f16 = p.q.type == KV_F16;
#pragma unroll 1
            for (int i0 = 0; i0 < 16; i0 += B) {
                const int in = all_rows - row0 - t * KE_M - ra - i0;  // rows there are (q_len is not known yet)
                uint32_t  u[B][E];  // F32 values, or 16-bit pairs in the first half
                if (p.q.vec) {
#pragma unroll
                    for (int i = 0; i < B; i++) {
                        const char * src = reinterpret_cast<const char *>(__shfl_sync(0xffffffffu, al, i0 + i));
                        if (E == 4) {
                            uint4 w = make_uint4(0, 0, 0, 0);
                            if (i < in && f32) {
                                w = *reinterpret_cast<const uint4 *>(src + lane * 16);
                            } else if (i < in) {
                                const uint2 v = *reinterpret_cast<const uint2 *>(src + lane * 8);
                                w.x = v.x, w.y = v.y;
                            }
                            u[i][0] = w.x, u[i][1] = w.y, u[i][E - 2] = w.z, u[i][E - 1] = w.w;
                        } else {
                            uint2 w = make_uint2(0, 0);
                            if (i < in && f32) {
                                w = *reinterpret_cast<const uint2 *>(src + lane * 8);
                            } else if (i < in) {
                                w.x = *reinterpret_cast<const uint32_t *>(src + lane * 4);
                            }
                            u[i][0] = w.x, u[i][1] = w.y;
                        }
                    }
                } else {
#pragma unroll
                    for (int i = 0; i < B; i++) {
                        const char * src = reinterpret_cast<const char *>(__shfl_sync(0xffffffffu, al, i0 + i));
#pragma unroll
                        for (int e = 0; e < E; e++) {
                            u[i][e] = i < in && f32 ? reinterpret_cast<const uint32_t *>(src)[e0 + e] : 0u;
                        }
                        if (i < in && !f32) {
#pragma unroll
                            for (int e = 0; e < E; e += 2) {
                                u[i][e / 2] = reinterpret_cast<const uint16_t *>(src)[e0 + e] | (uint32_t) reinterpret_cast<const uint16_t *>(src)[e0 + e + 1] << 16;
                            }
                        }
                    }
                }
                float    x[B][E], mine_f = 0.0f;
                uint32_t top[B];
#pragma unroll
                for (int i = 0; i < B; i++) {
                    top[i] = 0;
#pragma unroll
                    for (int e = 0; e < E; e += 2) {
                        const float2 a = h2_to_f2(u[i][e / 2]), b = bf2_to_f2(u[i][e / 2]);
                        x[i][e]     = f32 ? __uint_as_float(u[i][e]) : f16 ? a.x : b.x;
                        x[i][e + 1] = f32 ? __uint_as_float(u[i][e + 1]) : f16 ? a.y : b.y;
                        top[i]      = max(top[i], max(__float_as_uint(x[i][e]) & 0x7fffffffu, __float_as_uint(x[i][e + 1]) & 0x7fffffffu));
                    }
                }
#pragma unroll
                for (int i = 0; i < B; i++) {
                    top[i] = __reduce_max_sync(0xffffffffu, top[i]);
                }
#pragma unroll
                for (int i = 0; i < B; i++) {
                    // the largest element goes to [2^14, 2^15), the upper end of F16's range: an element keeps F16's 11 bits
                    // down to 2^-28 of it, and its remainder another 11 to 2^-17.  (Rows below 2^-112, where the power would not be
                    // a number, stay that much lower.)  A row with an infinity or NaN gives NaN
                    const bool  odd = top[i] >= 0x7f800000u;
                    const int   ex  = (top[i] == 0 || odd ? 0 : max((int) (top[i] >> 23) - 127, -112)) - 14;
                    const float dn  = __uint_as_float((uint32_t) (127 - ex) << 23);
                    mine_f          = lane == i ? (odd ? NAN : __uint_as_float((uint32_t) (127 + ex) << 23)) : mine_f;
                    uint32_t w[E / 2], v[E / 2];
#pragma unroll
                    for (int e = 0; e < E; e += 2) {
                        const float a = odd ? 0.0f : x[i][e] * dn, b = odd ? 0.0f : x[i][e + 1] * dn;
                        w[e / 2] = ke_pack(a, b);
                        const float2 f = h2_to_f2(w[e / 2]);
                        v[e / 2]       = ke_pack(a - f.x, b - f.y);
                    }
                    char * at = to + (ra + i0 + i) * 128 + ((((e0 % 64) / 8) ^ i) << 4);  // ra + i0: a multiple of 8
                    if (E == 4) {
                        *reinterpret_cast<uint2 *>(at) = make_uint2(w[0], w[E / 2 - 1]);
                        if (QP == 2) {
                            *reinterpret_cast<uint2 *>(at + L::QT) = make_uint2(v[0], v[E / 2 - 1]);
                        }
                    } else {
                        *reinterpret_cast<uint32_t *>(at) = w[0];
                        if (QP == 2) {
                            *reinterpret_cast<uint32_t *>(at + L::QT) = v[0];
                        }
                    }
                }
                if (lane < B) {
                    factors[t * KE_M + ra + i0 + lane] = mine_f * (CAP ? p.scale / p.softcap : p.scale * LOG2E);
                }
            }
            fence_proxy_async_smem();
            dn_mbar_arrive(&bar[KB_QREADY + t]);
        };
        // (a tile has 256 arrivals: two halves of a quadrant's rows by a warp each, or by one warp twice)
        stage_q(quad * 32 + (!TWO && wg == 3 ? 16 : 0));
        if (TWO) {
            stage_q(quad * 32 + 16);
        }
        if (!TWO && wg == 3) {
            // =================================================== O in registers
            float acc[D];
#pragma unroll
            for (int e = 0; e < D; e++) {
                acc[e] = 0.0f;
            }
            bool ok = true;
            for (int j = 0; j < tiles; j++) {
                if (!dn_wait_warp(&bar[KB_GROW + (j & 3)], (uint32_t) ((j >> 2) & 1), deadline) ||
                    !dn_wait_warp(&bar[KB_OFULL + (j & 1)], (uint32_t) ((j >> 1) & 1), deadline)) {
                    ok = false;
                    break;
                }
                tc_fence_after();
                const float g = grows[(j & 3) * KE_M + r];
#pragma unroll
                for (int c = 0; c < D / 32; c++) {
                    uint32_t o[32];
                    tmem_ld32(o_col + (uint32_t) ((j & 1) * D + c * 32), o);
                    tmem_ld_wait_tie(o);
#pragma unroll
                    for (int e = 0; e < 32; e++) {
                        acc[c * 32 + e] = fmaf(acc[c * 32 + e], g, __uint_as_float(o[e]));
                    }
                }
                tc_fence_before();
                dn_mbar_arrive(&bar[KB_OFREE + (j & 1)]);
            }
            // Q's shared memory takes the result: KB_LAST follows QREADY, KB_DONE the last product
            if (rows > 0) {
                if (!dn_wait_warp(&bar[KB_LAST], 0, deadline) || !dn_wait_warp(&bar[KB_DONE], 0, deadline)) {
                    ok = false;
                }
                if (!ok) {
                    atomicExch(abort_f, 1);
                }
                const float inv = parts > 1 ? 1.0f : grows[4 * KE_M + r], up = parts > 1 ? 1.0f : grows[5 * KE_M + r];
#pragma unroll
                for (int c = 0; c < D / 32; c++) {
                    uint32_t o[32];
#pragma unroll
                    for (int e = 0; e < 32; e++) {
                        o[e] = __float_as_uint(ok ? acc[c * 32 + e] * inv * up : 0.0f);
                    }
                    if (parts > 1) {
                        give(c, o);
                    } else {
                        stage_cols(c, o);
                    }
                }
                bool mine_too = true;
                if (parts > 1) {
                    mine_too = arrive();
                    if (mine_too) {
                        join();
                    }
                }
                if (mine_too) {
                    store_rows();
                }
            }
        } else if (tile_rows > 0) {
            if (!dn_wait_warp(&bar[KB_QREADY + t], 0, deadline)) {
                atomicExch(abort_f, 1);
            }
            // a row of NaN (its Q is 0) is taken like the others, and made NaN at the end if it has seen a key
            const float * its    = factors + t * KE_M + r;
            const float   factor = *its != *its ? 1.0f : *its;
            const int  rw    = row0 + t * KE_M + r;
            const bool live  = r < tile_rows;
            const int  my_q  = (int) kv8_div((uint32_t) rw, p.ratio_inv);
            const int  lim   = !live ? 0x7fffffff : (p.causal ? n - (nq - 1 - my_q) : n) - before;  // keys of this row
            const int  warp_lim = (int) __reduce_min_sync(0xffffffffu, (unsigned) max(lim, 0));
            float      m = -INFINITY, l = 0.0f, R = -INFINITY;
            bool       ok = true;
            for (int j = 0; j < tiles; j++) {
                const int      buf   = TWO ? t : j & 1, phase = TWO ? j : j >> 1;
                const uint32_t s_col = tmem + tl + (uint32_t) (buf * KE_N);
                if (!dn_wait_warp(&bar[KB_SCALES + (j & 3)], (uint32_t) ((j >> 2) & 1), deadline) ||
                    !dn_wait_warp(&bar[KB_SFULL + buf], (uint32_t) (phase & 1), deadline)) {
                    ok = false;
                    break;
                }
                tc_fence_after();
                const float4 * sc  = scales + (j & 3) * 8;
                const int      left = lim - j * KE_N;  // columns that the row sees
                if (CAP) {
                    // s = cap * tanh(S * factor * a), written back; the pass below takes it as it is
#pragma unroll 1
                    for (int c = 0; c < 4; c++) {
                        uint32_t v[32];
                        tmem_ld32(s_col + (uint32_t) (c * 32), v);
                        tmem_ld_wait_tie(v);
                        const float a0 = factor * sc[2 * c].x, a1 = factor * sc[2 * c + 1].x, cap = p.softcap * LOG2E;
#pragma unroll
                        for (int e = 0; e < 32; e++) {
                            v[e] = __float_as_uint(cap * tanhf(__uint_as_float(v[e]) * (e < 16 ? a0 : a1)));
                        }
                        tmem_st32(s_col + (uint32_t) (c * 32), v);
                    }
                    tmem_st_wait();
                }
                bool whole = j * KE_N + KE_N <= warp_lim;  // every row of the warp sees every column
                bool plain = !CAP;                         // s = S * factor * a, with all of these positive
#pragma unroll
                for (int g = 0; g < 8; g++) {
                    whole &= sc[g].w != 0.0f;
                    plain &= !(factor * sc[g].x <= 0.0f);
                }
                plain = __all_sync(0xffffffffu, plain);
                // The weights are taken with the maxima as they are (only a row's first tile has none), and the maxima found
                // and the weights taken again where a group's sum shows that one could leave F16's range
                // - by the rows that need it: no row's result depends on its neighbours'
                bool     need = m == -INFINITY || R == -INFINITY, full = __any_sync(0xffffffffu, need), fresh = false;
                float    grow = 1.0f, lsum, ms;
                uint32_t pk[KE_N / 2], pl[PP == 2 ? KE_N / 2 : 1];
#pragma unroll 1
                for (;;) {
                    uint32_t sr[KE_N];
#pragma unroll
                    for (int c = 0; c < 4; c++) {
                        tmem_ld32(s_col + (uint32_t) (c * 32), &sr[c * 32]);
                    }
#pragma unroll
                    for (int c = 0; c < 4; c++) {
                        tmem_ld_wait_tie(&sr[c * 32]);
                    }
                    if (!CAP && !plain) {
#pragma unroll
                        for (int e = 0; e < KE_N; e++) {
                            sr[e] = __float_as_uint(__uint_as_float(sr[e]) * (factor * sc[e >> 4].x));
                        }
                    }
                    if (!whole) {
#pragma unroll
                        for (int g = 0; g < 8; g++) {
                            const int lg = sc[g].w != 0.0f ? left : 0;
#pragma unroll
                            for (int e = 16 * g; e < 16 * g + 16; e++) {
                                sr[e] = e < lg ? sr[e] : 0xff800000u;
                            }
                        }
                    }
                    if (full) {  // the row's largest s, and the largest s + e over pages with a value scale
                        float top = m, rtop = R;
#pragma unroll
                        for (int g = 0; g < 8; g++) {
                            float a = __uint_as_float(sr[16 * g]), b = __uint_as_float(sr[16 * g + 1]);
#pragma unroll
                            for (int e = 16 * g + 2; e < 16 * g + 14; e += 4) {
                                a = fmax3(a, __uint_as_float(sr[e]), __uint_as_float(sr[e + 1]));
                                b = fmax3(b, __uint_as_float(sr[e + 2]), __uint_as_float(sr[e + 3]));
                            }
                            a    = fmaxf(fmax3(a, __uint_as_float(sr[16 * g + 14]), __uint_as_float(sr[16 * g + 15])), b);
                            a    = plain ? a * (factor * sc[g].x) : a;
                            top  = fmaxf(top, a);
                            rtop = sc[g].y != 0.0f ? fmaxf(rtop, a + sc[g].z) : rtop;
                        }
                        if (need) {
                            l *= m == top ? 1.0f : ex2(m - top);
                            grow = R == rtop ? 1.0f : ex2(R - rtop);
                            m = top, R = rtop, fresh = true;
                        }
                    }
                    ms = m == -INFINITY ? 0.0f : m;
                    const float    base = ms - (R == -INFINITY ? 0.0f : R) + KE_OFF;
                    const uint64_t nm = f2pack(-ms, -ms);
                    bool           high = false;
                    lsum                = 0.0f;
#pragma unroll
                    for (int g = 0; g < 8; g++) {
                        const float4   q  = sc[g];
                        const float    f  = ex2(fminf(base + q.z, 90.0f)) * q.y, a = plain ? factor * q.x : 1.0f;
                        const uint64_t f2 = f2pack(f, f), a2 = f2pack(a, a);
                        uint64_t       acc = 0ull;
#pragma unroll
                        for (int i = 8 * g; i < 8 * g + 8; i++) {
                            const uint64_t x2 = ffma2(f2pack(__uint_as_float(sr[2 * i]), __uint_as_float(sr[2 * i + 1])), a2, nm);
                            uint64_t       w2;
                            float          x, y;
                            if (PP == 1 && (i & 7) < KE_EMU) {
                                // over a stale maximum x has no bound, and the polynomial's exponent field would wrap
                                f2unpack(x2, x, y);
                                w2 = exp2_poly2(f2pack(fminf(x, 127.0f), fminf(y, 127.0f)));
                            } else {
                                f2unpack(x2, x, y);
                                w2 = f2pack(ex2(x), ex2(y));
                            }
                            acc = fadd2(acc, w2);
                            const uint64_t p2 = fmul2(w2, f2);
                            f2unpack(p2, x, y);
                            pk[i] = ke_pack(x, y);
                            if (PP == 2) {
                                const float2 b = h2_to_f2(pk[i]);
                                f2unpack(ffma2(f2pack(b.x, b.y), f2pack(-1.0f, -1.0f), p2), x, y);
                                pl[i] = ke_pack(x, y);
                            }
                        }
                        float x, y;
                        f2unpack(acc, x, y);
                        x += y;
                        lsum += x;
                        // the sum bounds every weight of the group; NaN and infinities fail the comparison below
                        high |= !(x * fabsf(f) <= 32768.0f);
                    }
                    // (and where it leaves F32's: value scales near 2^-126 would let a sum grow that far with P still small)
                    need = (high || !(lsum <= 0x1p100f)) && !fresh;
                    if (!__any_sync(0xffffffffu, need)) {
                        break;
                    }
                    full = true;
                }
                l += lsum + (ms - ms);  // a score of +inf: NaN
                if (!TWO) {
                    grows[(j & 3) * KE_M + r] = grow;
                    dn_mbar_arrive(&bar[KB_GROW + (j & 3)]);
                }
                tmem_st32(s_col, &pk[0]);
                tmem_st32(s_col + 32, &pk[32]);
                if (PP == 2) {
                    tmem_st32(s_col + 64, &pl[0]);
                    tmem_st32(s_col + 96, &pl[PP == 2 ? 32 : 0]);
                }
                // PV(j - 1) is complete: QK(j) was issued after it
                if (TWO && j > 0 && __any_sync(0xffffffffu, grow != 1.0f)) {
#pragma unroll 1
                    for (int c = 0; c < D / 32; c++) {
                        uint32_t o[32];
                        tmem_ld32(o_col + (uint32_t) (c * 32), o);
                        tmem_ld_wait_tie(o);
#pragma unroll
                        for (int e = 0; e < 32; e++) {
                            o[e] = __float_as_uint(__uint_as_float(o[e]) * grow);
                        }
                        tmem_st32(o_col + (uint32_t) (c * 32), o);
                    }
                }
                tmem_st_wait();
                tc_fence_before();
                dn_mbar_arrive(&bar[KB_PREADY + buf]);
            }
            l = *its != *its && m != -INFINITY ? NAN : l;
            // O (units of 2^(R - KE_OFF)) over the sum (2^m); rows without keys, and without a value scale, are 0
            const float inv = l != 0.0f ? (1.0f / (1 << KE_OFF)) / l : 0.0f, up = R == -INFINITY ? 0.0f : ex2(R - m);
            if (!TWO) {
                if (!ok) {
                    atomicExch(abort_f, 1);
                }
                grows[4 * KE_M + r] = inv, grows[5 * KE_M + r] = up;
                if (parts > 1) {
                    give_state(m, l, R);
                    __threadfence();  // the summing threads' arrival speaks for these too
                }
                dn_mbar_arrive(&bar[KB_LAST]);
            }
            if (TWO) {
            bool have = ok && tiles > 0;
            if (have) {
                have = dn_wait_warp(&bar[KB_OFULL + t], 0, deadline);
                tc_fence_after();
            }
            // Q's shared memory takes the result: every product has to be done
            if (!dn_wait_warp(&bar[KB_DONE], 0, deadline) || (!have && tiles > 0)) {
                atomicExch(abort_f, 1);
                have = false;
            }
#pragma unroll 1
            for (int c = 0; c < D / 32; c++) {
                uint32_t o[32];
                if (have) {
                    tmem_ld32(o_col + (uint32_t) (c * 32), o);
                    tmem_ld_wait_tie(o);
                } else {
#pragma unroll
                    for (int e = 0; e < 32; e++) {
                        o[e] = 0u;
                    }
                }
#pragma unroll
                for (int e = 0; e < 32; e++) {
                    o[e] = __float_as_uint(have ? __uint_as_float(o[e]) * (parts > 1 ? 1.0f : inv) * (parts > 1 ? 1.0f : up) : 0.0f);
                }
                if (parts > 1) {
                    give(c, o);
                } else {
                    stage_cols(c, o);
                }
            }
            bool mine_too = true;
            if (parts > 1) {
                give_state(m, l, R);
                mine_too = arrive();
                if (mine_too) {
                    join();
                }
            }
            if (mine_too) {
                store_rows();
            }
            }
        }
    }

    tc_fence_before();
    __syncthreads();
    if (warp == 4) {
        tc_fence_after();
        tmem_dealloc(tmem, KE_TMEM);
    }
    if (tid == 0 && *abort_f) {
        kv8_report(p.status, ST_TIMEOUT);
        atomicExch(&p.status[1], blockIdx.x);
    }
}

namespace {

template <int D, int QP, int PP, bool TWO, bool CAP>
cudaError_t launch_one(const Kv8AttnParams & p, cudaStream_t stream) {
    auto             kern = kv8_dense_kernel<D, QP, PP, TWO, CAP>;
    static Kv8Once   once;
    static const int regs = [&] {
        cudaFuncAttributes a{};
        return cudaFuncGetAttributes(&a, kern) == cudaSuccess ? a.numRegs : 0;
    }();
    // the register split draws on what the launch gives: another count would wait for registers that never come
    if (regs != KE_REGS_LAUNCH) {
        return cudaErrorInvalidConfiguration;
    }
    constexpr int   smem = KeSmem<D, QP, TWO>::TOTAL, step = TWO ? 256 : 128;
    const int64_t   rows = (int64_t) p.ratio * p.n_q, ctas = (rows + step - 1) / step * p.c.n_head_kv * p.t.n_seq * p.parts;
    const cudaError_t e  = once.smem(kern, smem);
    return e != cudaSuccess ? e : kv8_launch(kern, dim3((unsigned) ctas), KE_THREADS, smem, stream, p);
}

template <int D, bool CAP>
cudaError_t launch_d(const Kv8AttnParams & p, cudaStream_t stream) {
    if (p.o.type == KV_F32) {
        return launch_one<D, 2, 2, false, CAP>(p, stream);
    }
    if (p.o.type == KV_F16) {
        return launch_one<D, 1, 2, false, CAP>(p, stream);
    }
    return kv8_dense_tile(p) == KE_M ? launch_one<D, 1, 1, false, CAP>(p, stream) : launch_one<D, 1, 1, true, CAP>(p, stream);
}

}  // namespace

int kv8_dense_parts(int64_t items, int64_t tokens, int sms) {
    return (int) std::max<int64_t>(1, std::min<int64_t>({ sms / items, (tokens + KE_N * KE_PART - 1) / (KE_N * KE_PART), KE_PARTS }));
}

size_t kv8_dense_part_bytes(int D, int64_t items, int tile, int parts) {
    return parts > 1 ? (size_t) (items * parts) * (size_t) tile * (size_t) (D + 4) * 4 : 0;
}

int kv8_dense_tile(const Kv8AttnParams & p) {
    return p.o.type == KV_BF16 && (int64_t) p.t.max_pages * p.c.P <= KE_LONG ? 2 * KE_M : KE_M;
}

cudaError_t launch_kv8_dense(const Kv8AttnParams & p, cudaStream_t stream) {
    if (p.c.D == 64) {
        return p.softcap > 0.0f ? launch_d<64, true>(p, stream) : launch_d<64, false>(p, stream);
    }
    return p.softcap > 0.0f ? launch_d<128, true>(p, stream) : launch_d<128, false>(p, stream);
}

}  // namespace mm3fa
