// tree_attn_sm100.cu - attention of a tree of drafted tokens over a 16-bit slab cache on the 5th-generation tensor cores
// (tcgen05 + TMEM), sm_100a.
//
// Rows of a unit (sequence, kv head) are (node, head of the group) pairs in that order; a block has 128 of them, so the
// query heads of a kv head and the nodes share each K/V tile of 128 keys.  All CTAs (one per SM) are RB = blocks of a
// unit beside one another: groups of RB CTAs, each with one block, walk the same keys at the same time, so a K/V
// tile comes from HBM once.
//
// Split.  The tiles of all units are one line, in the order of sequence and kv head, and each group takes an equal piece of
// it, found on the device from the lengths: a long sequence is cut over many groups, short ones are several to a
// group, and no group waits for another.  (A group's piece may so have parts of two units, and whole ones between.)
// A part of a unit leaves O, m and l in the workspace, and a second kernel joins the parts in their order: by the last
// CTA to arrive, one SM of 148 would read all parts of a unit (25 us for 9 parts of 96 rows, at one SM's bandwidth).
// That kernel is left out where the slab is too short for a part.
//
// Most of the code runs once in a CTA, and its first run costs what the instruction cache costs: what does not feed the
// tensor core is in rolled loops or functions.
//
// 384 threads:
//   warp 0       TMA: K and V tiles through one ring, in the order in which the products take them
//   warp 1       TMEM allocation and every tcgen05.mma: QK(j + 1), then P V(j), P in TMEM over S
//   warps 2, 3   the V rows of tiles that hold nodes: those behind the last node become zero, and so do elements that are
//                no numbers (their weight may be 0; who sees such a node gets them added at the end)
//   warpgroups 1, 2   softmax of the even and the odd tiles, one row per thread, and the sum of their P V in registers:
//                two streams with maxima and sums of their own, joined at the piece's end
//
// Numerics.  q is brought to [2^14, 2^15) at its row's largest element by a power of two where the cache is F16, and rounded
// to the cache's type; where the result is F32, or q has another type than the cache, the remainder is a second operand, and
// so is that of the weights (PARTS 2; the remainder's product runs first, where the accumulator is small).  The tensor core
// truncates what it adds to an accumulator, up to 2^-23 of it in each step of 16 keys, always towards zero: every tile's
// P V starts afresh and is added in registers, rounded to nearest.
#include "fa_decode.cuh"
#include "tc_sm100.cuh"
#include "tree.cuh"

#include <algorithm>

namespace mm3fa {

namespace {

constexpr int TS_THREADS = 384;
constexpr int TS_M       = 128;  // rows of a block
constexpr int TS_N       = 128;  // keys of a tile
constexpr int TS_TMEM    = 512;  // columns: S of two tiles, P V of two tiles
constexpr int TS_OFF     = 14;   // weights are held times 2^14: F16 keeps 11 bits of one down to 2^-28 of the largest
constexpr int TJ_ROWS    = 8;    // rows of a joining CTA
constexpr int TS_REGS_LAUNCH  = 168;  // 65536 / 384, a multiple of 8
constexpr int TS_REGS_SOFTMAX = 208;  // 2 x 208 + 88 = 3 x 168
constexpr int TS_REGS_ISSUE   = 88;
static_assert(2 * TS_REGS_SOFTMAX + TS_REGS_ISSUE <= 3 * TS_REGS_LAUNCH, "more registers than the launch has");
constexpr int TS_SPACE = 256;  // bytes of the workspace before the list of units in parts
constexpr int TS_LEAST = 2;    // tiles of a part, at least: it costs about as much as a tile

template <int D, int PARTS>
struct TsSmem {
    static constexpr int HALVES = D / 64;  // 128-byte column blocks
    static constexpr int QT     = HALVES * TS_M * 128;
    static constexpr int KT     = HALVES * TS_N * 128;
    static constexpr int NS     = D == 128 ? (PARTS == 2 ? 4 : 5) : 8;  // tiles in the ring
    static constexpr int XCH    = 2 * TS_M * 32 * 4;                    // exchange of the two streams' sums, in Q's place
    static constexpr int Q_ALL  = PARTS * QT > XCH ? PARTS * QT : XCH;
    static constexpr int OFF_Q    = 0;
    static constexpr int OFF_RING = OFF_Q + Q_ALL;
    static constexpr int OFF_ANC  = OFF_RING + NS * KT;           // [TREE_MAX][TREE_MAX / 32] bits
    static constexpr int OFF_PAR  = OFF_ANC + TREE_MAX * (TREE_MAX / 32) * 4;
    static constexpr int OFF_F    = OFF_PAR + TREE_MAX * 4;       // [row] factors
    static constexpr int OFF_ML   = OFF_F + TS_M * 4;             // [stream][row] (m, l)
    static constexpr int OFF_BAR  = OFF_ML + 2 * TS_M * 8;
    static constexpr int OFF_MISC = OFF_BAR + 48 * 8;
    static constexpr int TOTAL    = OFF_MISC + 256 + 1024;        // + alignment
};
static_assert(TsSmem<128, 1>::TOTAL <= 232448 && TsSmem<128, 2>::TOTAL <= 232448 && TsSmem<64, 2>::TOTAL <= 232448, "shared memory");

enum : int {
    TB_FULL   = 0,   // [8] TMA
    TB_EMPTY  = 8,   // [8] products
    TB_SFULL  = 16,  // [2]
    TB_PREADY = 18,  // [2] 128 softmax threads
    TB_OFULL  = 20,  // [2]
    TB_OFREE  = 22,  // [2] 128 softmax threads
    TB_QREADY = 24,  // 256
    TB_LOOK   = 25,  // warp 1: a V tile with nodes is there
    TB_FIX    = 26,  // 64 threads of warps 2, 3: it can be taken
    TB_DONE   = 27,
    TB_COUNT  = 28,
};

__host__ __device__ constexpr uint32_t ts_arrivals(int b) {
    return b == TB_QREADY ? 256u : b == TB_FIX ? 64u : ((b >= TB_PREADY && b < TB_OFULL) || (b >= TB_OFREE && b < TB_QREADY)) ? 128u : 1u;
}

// kind::f16 instruction descriptor: F16 x F16 or BF16 x BF16 -> F32, M = 128
__host__ __device__ constexpr uint32_t ts_idesc(bool bf16, int n, bool b_mn_major) {
    return (1u << 4) | ((bf16 ? 1u : 0u) << 7) | ((bf16 ? 1u : 0u) << 10) | ((b_mn_major ? 1u : 0u) << 16) | ((uint32_t) (n >> 3) << 17) |
           ((uint32_t) (TS_M >> 4) << 24);
}

__device__ __forceinline__ void ts_load(void * dst, const CUtensorMap * tm, int c0, int c1, int c2, int c3, uint64_t * bar) {
    asm volatile(
        "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], "
        "[%6];" ::"r"(smem_addr(dst)),
        "l"(reinterpret_cast<uint64_t>(tm)), "r"(c0), "r"(c1), "r"(c2), "r"(c3), "r"(smem_addr(bar))
        : "memory");
}

__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t * r) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(taddr),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]),
        "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
        : "memory");
}

__device__ __forceinline__ void softmax_barrier() {  // the 256 threads of both streams
    asm volatile("bar.sync 1, 256;" ::: "memory");
}

template <bool BF16>
__device__ __forceinline__ uint32_t ts_pack(float lo, float hi) {
    if (BF16) {
        const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
        return *reinterpret_cast<const uint32_t *>(&v);
    }
    const __half2 v = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t *>(&v);
}

// the same, rounded towards zero
template <bool BF16>
__device__ __forceinline__ uint32_t ts_pack_rz(float lo, float hi) {
    uint32_t u;
    if (BF16) {
        asm("cvt.rz.bf16x2.f32 %0, %1, %2;" : "=r"(u) : "f"(hi), "f"(lo));
    } else {
        asm("cvt.rz.f16x2.f32 %0, %1, %2;" : "=r"(u) : "f"(hi), "f"(lo));
    }
    return u;
}

// each of two numbers that are not negative, or the smallest positive one
template <bool BF16>
__device__ __forceinline__ uint32_t ts_positive(uint32_t u) {
    return __vmaxu2(u, BF16 ? 0x00800080u : 0x00010001u);
}

template <bool BF16>
__device__ __forceinline__ float2 ts_unpack(uint32_t u) {
    return BF16 ? bf2_to_f2(u) : h2_to_f2(u);
}

// (functions of their own: see the instruction cache above)
__device__ __noinline__ float ts_tanh(float x) {
    return tanhf(x);
}

// elements [e0, e0 + E) of a row that is not aligned: F32, or 16-bit pairs
template <int E>
__device__ __noinline__ uint4 ts_load_elements(const char * row, bool f32, int e0) {
    uint32_t x[4] = { 0, 0, 0, 0 };
    if (f32) {
#pragma unroll
        for (int e = 0; e < E; e++) {
            x[e] = reinterpret_cast<const uint32_t *>(row)[e0 + e];
        }
    } else {
#pragma unroll
        for (int e = 0; e < E; e += 2) {
            x[e / 2] = reinterpret_cast<const uint16_t *>(row)[e0 + e] | (uint32_t) reinterpret_cast<const uint16_t *>(row)[e0 + e + 1] << 16;
        }
    }
    return make_uint4(x[0], x[1], x[2], x[3]);
}

// Floats of a part: O of its rows, then m and l of each; a multiple of 16 bytes.
__host__ __device__ constexpr int ts_slot_floats(int rows, int D) {
    return (rows * (D + 2) + 3) / 4 * 4;
}

// 4 values to elements [e, e + 4) of a row
__device__ __forceinline__ void ts_store4(char * row, int e, const float4 & f, int type, bool vec) {
    if (type == KV_F32) {
        float * o = reinterpret_cast<float *>(row) + e;
        if (vec) {
            *reinterpret_cast<float4 *>(o) = f;
        } else {
            o[0] = f.x, o[1] = f.y, o[2] = f.z, o[3] = f.w;
        }
        return;
    }
    const uint32_t a = type == KV_F16 ? ts_pack<false>(f.x, f.y) : ts_pack<true>(f.x, f.y);
    const uint32_t b = type == KV_F16 ? ts_pack<false>(f.z, f.w) : ts_pack<true>(f.z, f.w);
    uint16_t *     o = reinterpret_cast<uint16_t *>(row) + e;
    if (vec) {
        *reinterpret_cast<uint2 *>(o) = make_uint2(a, b);
    } else {
        o[0] = (uint16_t) a, o[1] = (uint16_t) (a >> 16), o[2] = (uint16_t) b, o[3] = (uint16_t) (b >> 16);
    }
}

// What the group that has a unit's first part leaves for the joining kernel.
struct TsJoin {
    int     s, h, parts, rows;  // parts 0: the group has no such unit
    int64_t part0, part1;       // where the first part and the second are, in floats; the others follow at even steps
};

// Key tiles of a sequence's units; 0 where none of its nodes counts.
struct TsSeq {
    int L, nodes, keys, tiles;
};

__device__ __forceinline__ TsSeq ts_seq(const TreeAttnParams & p, int s) {
    TsSeq q;
    q.nodes = tree_nodes(p.t, s % p.t.n_tree);
    q.L     = min(max(p.kv_len[s], 0), p.n_kv);
    q.keys  = q.nodes > 0 ? min(q.L + q.nodes, p.n_kv) : 0;
    q.tiles = (q.keys + TS_N - 1) / TS_N;
    return q;
}

// The line of W tiles in G even pieces, piece g from `at(g)` on.  A border closer than TS_LEAST tiles to a unit's start or end
// goes there, so that no part of a unit has less.
struct TsLine {
    int W, G, each, more;  // `more` pieces have a tile more than `each`

    __device__ __forceinline__ TsLine(int W_, int groups) : W(W_), G(max(1, min(groups, W_ / TS_LEAST))) {
        each = W / G;
        more = W - each * G;
    }

    __device__ __forceinline__ int at(int g) const {
        return g * each + min(g, more);
    }

    // the last piece that starts at tile x or before
    __device__ __forceinline__ int last(int x) const {
        const int y = more * (each + 1);
        return min(G - 1, x < y ? x / (each + 1) : each > 0 ? more + (x - y) / each : G - 1);
    }

    // border x, of a unit of n tiles that starts at `first` and holds x
    static __device__ __forceinline__ int border(int x, int first, int n) {
        return x - first < TS_LEAST ? first : first + n - x < TS_LEAST ? first + n : x;
    }
};

// The pieces of a group: tiles [a, b) of unit (s, h), one after another.  Every role walks them by itself.
struct TsPieces {
    const TreeAttnParams & p;
    int                    s, first, x, end;  // first: of sequence s on the line of tiles; end: before its move to a border
    TsSeq                  q;
    int                    h, a, b, unit;     // unit: where the unit starts

    __device__ __forceinline__ TsPieces(const TreeAttnParams & p_, int s_, int first_, int x_, int end_)
        : p(p_), s(s_), first(first_), x(x_), end(end_), q{ 0, 0, 0, 0 }, h(0), a(0), b(0), unit(0) {
        if (x < end) {
            q = ts_seq(p, s);
            const int u = first + (x - first) / q.tiles * q.tiles;
            x           = TsLine::border(x, u, q.tiles);
        }
    }

    // the next piece that has rows in block rb
    __device__ __forceinline__ bool next(int rb) {
        while (x < end) {
            const int all = q.tiles * p.n_head_kv;
            if (x - first >= all) {
                first += all;
                q = ts_seq(p, ++s);
                continue;
            }
            if (q.nodes * p.ratio <= rb * TS_M) {  // (this block is empty: on to the next sequence)
                x = first + all;
                continue;
            }
            h    = (x - first) / q.tiles;
            unit = first + h * q.tiles;
            a    = x - unit;
            b    = unit + q.tiles <= end ? q.tiles : TsLine::border(end, unit, q.tiles) - unit;
            if (b <= a) {
                return false;
            }
            x = unit + b;
            return true;
        }
        return false;
    }
};

template <int D, bool BF16, int PARTS>
__global__ void __launch_bounds__(TS_THREADS, 1)
    tree_attn_tc_kernel(const __grid_constant__ CUtensorMap tmk, const __grid_constant__ CUtensorMap tmv, const TreeAttnParams p, int blocks,
                        int groups, int slot_rows) {
    using L          = TsSmem<D, PARTS>;
    constexpr int NS = L::NS;
    extern __shared__ __align__(16) char smem_raw[];
    char *     smem      = smem_raw + ((1024u - (smem_addr(smem_raw) & 1023u)) & 1023u);
    uint64_t * bar       = reinterpret_cast<uint64_t *>(smem + L::OFF_BAR);
    uint32_t * misc      = reinterpret_cast<uint32_t *>(smem + L::OFF_MISC);
    uint32_t * tmem_slot = misc;
    int *      abort_f   = reinterpret_cast<int *>(misc + 1);
    int *      start_s   = reinterpret_cast<int *>(misc + 3);
    int *      line      = reinterpret_cast<int *>(misc + 4);       // the whole line's tiles, the first one of start_s
    int *      dirty     = reinterpret_cast<int *>(misc + 8);       // a V row of the piece's nodes held what is no number
    int *      sums      = reinterpret_cast<int *>(misc + 16);      // [12] warps' counts
    float *    factors   = reinterpret_cast<float *>(smem + L::OFF_F);
    float2 *   ml        = reinterpret_cast<float2 *>(smem + L::OFF_ML);
    uint32_t * anc       = reinterpret_cast<uint32_t *>(smem + L::OFF_ANC);
    int *      par       = reinterpret_cast<int *>(smem + L::OFF_PAR);

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, wg = warp >> 2;
    if (tid == 0) {
        for (int i = 0; i < TB_COUNT; i++) {
            mbar_init(&bar[i], ts_arrivals(i));
        }
        *abort_f = 0, *start_s = 0, line[1] = 0, *dirty = 0;
        fence_mbar_init();
    }
    if (warp == 1) {
        tmem_alloc(tmem_slot, TS_TMEM);
        tmem_relinquish();
    }
    kv8_dep_wait();
    const uint64_t deadline = global_timer_ns() + p.timeout_ns;

    // ---- the group's piece of the line of tiles
    const int group = (int) blockIdx.x / blocks, rb = (int) blockIdx.x % blocks;
    TsJoin *  join  = reinterpret_cast<TsJoin *>(reinterpret_cast<char *>(p.status) + TS_SPACE) + blockIdx.x;
    if (tid == 0) {
        join->parts = 0;
    }
    {
        // each thread sums some sequences' tiles of one kv head; all tiles are fewer than 2^30 (checked by the host)
        const int each = (p.n_seq + TS_THREADS - 1) / TS_THREADS, s0 = min(tid * each, p.n_seq), s1 = min(s0 + each, p.n_seq);
        int       mine = 0;
        for (int s = s0; s < s1; s++) {
            mine += ts_seq(p, s).tiles;
        }
        int upto = mine;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const int y = __shfl_up_sync(0xffffffffu, upto, d);
            upto += lane >= d ? y : 0;
        }
        if (lane == 31) {
            sums[warp] = upto;
        }
        tc_fence_before();
        __syncthreads();
        tc_fence_after();
        int before = 0, all = 0;
#pragma unroll
        for (int w = 0; w < TS_THREADS / 32; w++) {
            before += w < warp ? sums[w] : 0;
            all += sums[w];
        }
        const TsLine ln(all * p.n_head_kv, groups);
        const int    from = ln.at(group);
        int          at   = (before + upto - mine) * p.n_head_kv;
        if (group < ln.G && from >= at && from < at + mine * p.n_head_kv) {  // it starts among this thread's
            int s = s0;
            for (;; s++) {
                const int n = ts_seq(p, s).tiles * p.n_head_kv;
                if (from < at + n) {
                    break;
                }
                at += n;
            }
            *start_s = s, line[1] = at;
        }
        if (tid == 0) {
            line[0] = ln.W;
        }
        __syncthreads();
    }
    const uint32_t tmem = *tmem_slot;
    const TsLine   ln(line[0], groups);
    TsPieces       it(p, *start_s, line[1], group < ln.G ? ln.at(group) : ln.W, group < ln.G ? ln.at(group + 1) : ln.W);

    if (wg == 0) {
        regs_dec<TS_REGS_ISSUE>();
        bool ok = true;
        if (warp == 0) {
            // =================================================== TMA
            if (lane == 0) {
                uint32_t c = 0;
                auto     load = [&](const CUtensorMap * tm, int tile) {
                    const int slot = (int) (c % NS);
                    if (ok && c >= (uint32_t) NS && !mbar_wait_bounded(&bar[TB_EMPTY + slot], (c / NS - 1) & 1, deadline)) {
                        ok = false;
                    }
                    if (ok) {
                        mbar_arrive_expect_tx(&bar[TB_FULL + slot], (uint32_t) L::KT);
#pragma unroll
                        for (int hf = 0; hf < L::HALVES; hf++) {
                            ts_load(smem + L::OFF_RING + slot * L::KT + hf * (TS_N * 128), tm, hf * 64, tile * TS_N, it.h, it.s, &bar[TB_FULL + slot]);
                        }
                        c++;
                    }
                };
                while (ok && it.next(rb)) {
                    load(&tmk, it.a);
                    for (int j = it.a; ok && j < it.b; j++) {
                        if (j + 1 < it.b) {
                            load(&tmk, j + 1);
                        }
                        load(&tmv, j);
                    }
                }
                if (!ok) {  // copies that are under way have to land
                    const uint64_t limit = global_timer_ns() + p.timeout_ns;
                    for (uint32_t i = c > (uint32_t) NS ? c - NS : 0; i < c; i++) {
                        mbar_wait_bounded(&bar[TB_FULL + i % NS], (i / NS) & 1, limit);
                    }
                }
            }
            __syncwarp();
        } else if (warp == 1) {
            // =================================================== products
            const uint32_t id_qk = ts_idesc(BF16, TS_N, false), id_pv = ts_idesc(BF16, D, true);
            const uint64_t q_d = sw128_desc(smem_addr(smem + L::OFF_Q), 16, 1024), k_d = sw128_desc(smem_addr(smem + L::OFF_RING), 16, 1024);
            const uint64_t v_d = sw128_desc(smem_addr(smem + L::OFF_RING), (uint32_t) (TS_N * 128), 1024);
            auto wait = [&](int b, uint32_t i) {
                if (ok && !dn_wait_warp(&bar[b], i & 1, deadline)) {
                    ok = false;
                }
                tc_fence_after();
            };
            uint32_t c = 0, tc = 0, fixes = 0, pieces = 0;
            auto     qk = [&](uint32_t t) {
                const int slot = (int) (c % NS), buf = (int) (t & 1);
                wait(TB_FULL + slot, c / NS);
#pragma unroll 1
                for (int part = PARTS - 1; part >= 0; part--) {
                    uint64_t qa = q_d + (uint64_t) ((part * L::QT) >> 4), kb = k_d + (uint64_t) ((slot * L::KT) >> 4);
#pragma unroll
                    for (int hf = 0; hf < L::HALVES; hf++) {
#pragma unroll
                        for (int k = 0; k < 4; k++) {
                            umma_f16(tmem + (uint32_t) (buf * TS_N), qa + (uint64_t) (2 * k), kb + (uint64_t) (2 * k), id_qk, PARTS - 1 - part + hf + k > 0 ? 1u : 0u);
                        }
                        qa += (TS_M * 128) >> 4, kb += (TS_N * 128) >> 4;
                    }
                }
                umma_commit(&bar[TB_EMPTY + slot]);
                umma_commit(&bar[TB_SFULL + buf]);
                c++;
            };
            while (it.next(rb)) {
                wait(TB_QREADY, pieces++);
                qk(tc);
                for (int j = it.a; j < it.b; j++, tc++) {
                    if (j + 1 < it.b) {
                        qk(tc + 1);
                    }
                    const int slot = (int) (c % NS), buf = (int) (tc & 1);
                    wait(TB_FULL + slot, c / NS);
                    const bool nodes = (j + 1) * TS_N > it.q.L;
                    if (nodes && lane == 0) {
                        dn_mbar_arrive(&bar[TB_LOOK]);
                    }
                    wait(TB_PREADY + buf, tc >> 1);
                    if (tc >= 2) {
                        wait(TB_OFREE + buf, (tc >> 1) - 1);
                    }
                    if (nodes) {
                        wait(TB_FIX, fixes++);
                    }
#pragma unroll 1
                    for (int part = PARTS - 1; part >= 0; part--) {
                        uint32_t a = tmem + (uint32_t) (buf * TS_N + part * 16);
                        uint64_t b = v_d + (uint64_t) ((slot * L::KT) >> 4);
#pragma unroll
                        for (int k = 0; k < 8; k++) {  // P of 32 keys: 16 columns, then 16 of its remainder
                            umma_f16_ts(tmem + 256u + (uint32_t) (buf * D), a + (uint32_t) ((k >> 1) * 16 * PARTS + (k & 1) * 8), b + (uint64_t) ((k * 16 * 128) >> 4),
                                        id_pv, PARTS - 1 - part + k > 0 ? 1u : 0u);
                        }
                    }
                    umma_commit(&bar[TB_EMPTY + slot]);
                    umma_commit(&bar[TB_OFULL + buf]);
                    c++;
                }
            }
            // every product issued has to be complete before TMEM and shared memory are given up
            umma_commit(&bar[TB_DONE]);
            dn_wait_warp(&bar[TB_DONE], 0, global_timer_ns() + p.timeout_ns);
        } else {
            // =================================================== V rows of tiles that hold nodes
            const int t64 = tid - 64;
            uint32_t  c = 0, fixes = 0;
            while (it.next(rb)) {
                const int n = it.b - it.a;
                for (int j = max(it.a, it.q.L / TS_N); j < it.b; j++) {
                    const uint32_t i    = c + (uint32_t) (2 * (j - it.a) + (j + 1 < it.b ? 2 : 1));  // its place in the ring's order
                    const int      slot = (int) (i % NS);
                    // (warp 1 has seen the tile land and keeps its place until it is looked at, so that the second wait
                    // finds the phase it names)
                    if (ok && (!dn_wait_warp(&bar[TB_LOOK], fixes & 1, deadline) || !dn_wait_warp(&bar[TB_FULL + slot], (i / NS) & 1, deadline))) {
                        ok = false;
                    }
                    char *    tile = smem + L::OFF_RING + slot * L::KT;
                    const int r0 = max(0, it.q.L - j * TS_N), end = it.q.keys - j * TS_N;
                    bool      odd = false;
                    for (int e = t64; e < (TS_N - r0) * 8 * L::HALVES; e += 64) {
                        const int r  = r0 + e / (8 * L::HALVES), ck = e % (8 * L::HALVES);
                        uint4 *   at = reinterpret_cast<uint4 *>(tile + (ck >> 3) * (TS_N * 128) + r * 128 + (ck & 7) * 16);
                        if (r >= end) {
                            *at = make_uint4(0, 0, 0, 0);
                            continue;
                        }
                        uint4              w    = *at;
                        constexpr uint32_t EXP  = BF16 ? 0x7f80u : 0x7c00u;
                        bool               here = false;
#pragma unroll
                        for (int k = 0; k < 4; k++) {
                            uint32_t & u = (&w.x)[k];
                            if ((u & EXP) == EXP) {
                                u &= 0xffff0000u, here = true;
                            }
                            if ((u >> 16 & EXP) == EXP) {
                                u &= 0xffffu, here = true;
                            }
                        }
                        if (here) {
                            *at = w;
                            odd = true;
                        }
                    }
                    if (odd) {
                        atomicExch(dirty, 1);
                    }
                    fence_proxy_async_smem();
                    dn_mbar_arrive(&bar[TB_FIX]);
                    fixes++;
                }
                c += (uint32_t) (2 * n);
            }
        }
        if (!ok) {
            atomicExch(abort_f, 1);
        }
    } else {
        // ======================================================= softmax and sums
        regs_inc<TS_REGS_SOFTMAX>();
        const int      w = wg - 1, quad = warp & 3, r = quad * 32 + lane, row = rb * TS_M + r, own = tid - 128;
        const uint32_t tl    = (uint32_t) (quad * 32) << 16;
        const uint32_t s_col = tmem + tl + (uint32_t) (w * TS_N), o_col = tmem + tl + 256u + (uint32_t) (w * D);
        const int      my_node = row / p.ratio;
        const bool     cap = p.softcap > 0.0f;
        char *         qs  = smem + L::OFF_Q;
        float4 *       xch = reinterpret_cast<float4 *>(smem + L::OFF_Q);
        uint32_t       tc = 0;
        bool           ok = true;
        auto           wait = [&](int b, uint32_t i) {
            if (ok && !dn_wait_warp(&bar[b], i & 1, deadline)) {
                ok = false;
            }
            tc_fence_after();
        };
        while (it.next(rb)) {
            const int  its_rows = min(it.q.nodes * p.ratio - rb * TS_M, TS_M);
            const bool live = r < its_rows, warp_live = quad * 32 < its_rows;
            const int  held = it.q.L, nodes = it.q.nodes;
            // ---- Q: 16 rows by each warp, all loads in flight, 8 rows at a time
            {
                constexpr int  E = D / 32, B = 8;
                const int      ra = (w * 4 + quad) * 16, e0 = lane * E, in = its_rows - ra;
                char *         to = qs + (e0 / 64) * (TS_M * 128) + ra * 128 + (e0 % 8) * 2;
                const float    sign = p.scale < 0.0f ? -1.0f : 1.0f, by = fabsf(cap ? p.scale / p.softcap : p.scale * LOG2E);
                // lane i: the address of row i
                const int      rl = rb * TS_M + ra + (lane & 15), nl = rl / p.ratio, hl = it.h * p.ratio + rl - nl * p.ratio;
                const uint64_t al = reinterpret_cast<uint64_t>(p.q.data + (int64_t) nl * p.q.nb1 + (int64_t) hl * p.q.nb2 + (int64_t) it.s * p.q.nb3);
                uint32_t       u[2][B][E];  // F32 values, or 16-bit pairs in the first half
                const bool     f32 = p.q.type == KV_F32, f16 = p.q.type == KV_F16;
#pragma unroll
                for (int i = 0; i < 2 * B; i++) {
                    const char * src = reinterpret_cast<const char *>(__shfl_sync(0xffffffffu, al, i));
                    uint32_t (&x)[E] = u[i / B][i % B];
#pragma unroll
                    for (int e = 0; e < E; e++) {
                        x[e] = 0u;
                    }
                    if (i < in && p.q.vec) {
                        if (E == 4 && f32) {
                            const uint4 f = *reinterpret_cast<const uint4 *>(src + lane * 16);
                            x[0] = f.x, x[1] = f.y, x[E - 2] = f.z, x[E - 1] = f.w;
                        } else if (E == 4 || f32) {
                            const uint2 f = *reinterpret_cast<const uint2 *>(src + lane * 8);
                            x[0] = f.x, x[1] = f.y;
                        } else {
                            x[0] = *reinterpret_cast<const uint32_t *>(src + lane * 4);
                        }
                    }
                }
#pragma unroll 1
                for (int half = 0; half < 2; half++) {
                    if (!p.q.vec) {  // by elements, a row after another
#pragma unroll
                        for (int i = 0; i < B; i++) {
                            const char * src = reinterpret_cast<const char *>(__shfl_sync(0xffffffffu, al, half * B + i));
                            if (half * B + i < in) {
                                const uint4 f = ts_load_elements<E>(src, f32, e0);
                                u[0][i][0] = f.x, u[0][i][1] = f.y;
                                if (E == 4) {
                                    u[0][i][E - 2] = f.z, u[0][i][E - 1] = f.w;
                                }
                            }
                        }
                    }
#pragma unroll
                    for (int i = 0; i < B; i++) {
                        float    x[E];
                        uint32_t top = 0;
#pragma unroll
                        for (int e = 0; e < E; e += 2) {
                            const float2 a = f16 ? h2_to_f2(u[0][i][e / 2]) : bf2_to_f2(u[0][i][e / 2]);
                            x[e]     = f32 ? __uint_as_float(u[0][i][e]) : a.x;
                            x[e + 1] = f32 ? __uint_as_float(u[0][i][e + 1]) : a.y;
                            top      = max(top, max(__float_as_uint(x[e]) & 0x7fffffffu, __float_as_uint(x[e + 1]) & 0x7fffffffu));
                        }
                        top = __reduce_max_sync(0xffffffffu, top);
                        // a row with an infinity or NaN gives NaN.  F16: the largest element goes to [2^14, 2^15)
                        const bool  odd = top >= 0x7f800000u;
                        const int   ex  = BF16 ? 0 : (top == 0 || odd ? 0 : max((int) (top >> 23) - 127, -112)) - 14;
                        const float dn  = __uint_as_float((uint32_t) (127 - ex) << 23) * sign;
                        uint32_t    hi[E / 2], lo[E / 2];
#pragma unroll
                        for (int e = 0; e < E; e += 2) {
                            const float a = odd ? 0.0f : x[e] * dn, b = odd ? 0.0f : x[e + 1] * dn;
                            hi[e / 2]      = ts_pack<BF16>(a, b);
                            const float2 f = ts_unpack<BF16>(hi[e / 2]);
                            lo[e / 2]      = ts_pack<BF16>(a - f.x, b - f.y);
                        }
                        char * at = to + (half * B + i) * 128 + ((((e0 % 64) / 8) ^ i) << 4);  // ra and B: multiples of 8
                        if (E == 4) {
                            *reinterpret_cast<uint2 *>(at) = make_uint2(hi[0], hi[E / 2 - 1]);
                            if (PARTS == 2) {
                                *reinterpret_cast<uint2 *>(at + L::QT) = make_uint2(lo[0], lo[E / 2 - 1]);
                            }
                        } else {
                            *reinterpret_cast<uint32_t *>(at) = hi[0];
                            if (PARTS == 2) {
                                *reinterpret_cast<uint32_t *>(at + L::QT) = lo[0];
                            }
                        }
                        if (lane == i) {
                            factors[ra + half * B + i] = odd ? NAN : __uint_as_float((uint32_t) (127 + ex) << 23) * by;
                        }
#pragma unroll
                        for (int e = 0; e < E; e++) {
                            u[0][i][e] = u[1][i][e];
                        }
                    }
                }
                fence_proxy_async_smem();
                dn_mbar_arrive(&bar[TB_QREADY]);
            }
            // ---- each node's ancestors, where the piece has tiles with nodes
            const bool tail = it.b * TS_N > held;
            if (tail) {
                if (own < nodes) {
                    par[own] = tree_parent(p.t, it.s % p.t.n_tree, own);
                }
                softmax_barrier();
                if (own < nodes) {
                    uint32_t * bits = anc + own * (TREE_MAX / 32);
#pragma unroll
                    for (int k = 0; k < TREE_MAX / 32; k++) {
                        bits[k] = 0;
                    }
                    for (int at = own; at >= 0; at = par[at]) {
                        bits[at >> 5] |= held + at < p.n_kv ? 1u << (at & 31) : 0u;
                    }
                }
            }
            softmax_barrier();  // (and all of Q's factors are there)
            const float    f0 = factors[r], factor = cap || f0 != f0 ? 1.0f : f0;
            const float    fcap = f0 != f0 ? 1.0f : f0;
            const uint32_t * bits = anc + min(my_node, TREE_MAX - 1) * (TREE_MAX / 32);
            // which of the 32 keys from k0 on the row sees
            auto seen = [&](int k0) -> uint32_t {
                const int o = k0 - held;  // in nodes
                if (o <= -32) {
                    return 0xffffffffu;
                }
                if (o >= TREE_MAX) {
                    return 0u;
                }
                if (o < 0) {
                    return (1u << -o) - 1u | bits[0] << -o;
                }
                const uint32_t lo = bits[o >> 5], hi = o + 32 < TREE_MAX ? bits[(o >> 5) + 1] : 0u;
                return __funnelshift_r(lo, hi, o & 31);
            };
            float m = -INFINITY, l = 0.0f, acc[D];
#pragma unroll
            for (int e = 0; e < D; e++) {
                acc[e] = 0.0f;
            }
            for (int j = it.a; j < it.b; j++, tc++) {
                if ((int) (tc & 1) != w) {
                    continue;
                }
                wait(TB_SFULL + w, tc >> 1);
                float g = 1.0f;
                if (warp_live) {
                    if (cap) {
#pragma unroll 1
                        for (int c = 0; c < 4; c++) {
                            uint32_t v[32];
                            tmem_ld32(s_col + (uint32_t) (c * 32), v);
                            tmem_ld_wait_tie(v);
#pragma unroll
                            for (int e = 0; e < 32; e++) {
                                v[e] = __float_as_uint(ts_tanh(__uint_as_float(v[e]) * fcap) * (p.softcap * LOG2E));
                            }
                            tmem_st32(s_col + (uint32_t) (c * 32), v);
                        }
                        tmem_st_wait();
                    }
                    const bool masked = (j + 1) * TS_N > held;
                    float      top = -INFINITY;
#pragma unroll 1
                    for (int c = 0; c < 4; c++) {
                        uint32_t v[32];
                        tmem_ld32(s_col + (uint32_t) (c * 32), v);
                        tmem_ld_wait_tie(v);
                        if (masked) {
                            const uint32_t see = live ? seen(j * TS_N + c * 32) : 0u;
#pragma unroll
                            for (int e = 0; e < 32; e++) {
                                v[e] = see >> e & 1u ? v[e] : 0xff800000u;
                            }
                        }
                        float a = __uint_as_float(v[0]), b = __uint_as_float(v[1]);
#pragma unroll
                        for (int e = 2; e < 30; e += 4) {
                            a = fmax3(a, __uint_as_float(v[e]), __uint_as_float(v[e + 1]));
                            b = fmax3(b, __uint_as_float(v[e + 2]), __uint_as_float(v[e + 3]));
                        }
                        top = fmax3(top, fmax3(a, __uint_as_float(v[30]), __uint_as_float(v[31])), b);
                    }
                    // (a factor of 0 makes a product with -inf no number)
                    const float mn = fmaxf(m, top == -INFINITY ? top : top * factor);
                    g = m == mn ? 1.0f : ex2(m - mn);
                    m = mn;
                    const float    nm = (m == -INFINITY ? 0.0f : -m) + (float) TS_OFF;
                    const uint64_t nm2 = f2pack(nm, nm), fa2 = f2pack(factor, factor);
                    uint64_t       sum2 = 0ull;
#pragma unroll 1
                    for (int c = 0; c < 4; c++) {
                        uint32_t v[32], hi[16], lo[PARTS == 2 ? 16 : 1];
                        tmem_ld32(s_col + (uint32_t) (c * 32), v);
                        tmem_ld_wait_tie(v);
                        const uint32_t see = !masked ? 0xffffffffu : live ? seen(j * TS_N + c * 32) : 0u;
#pragma unroll
                        for (int i = 0; i < 16; i++) {
                            float          x, y;
                            f2unpack(ffma2(f2pack(__uint_as_float(v[2 * i]), __uint_as_float(v[2 * i + 1])), fa2, nm2), x, y);
                            if (masked) {
                                x = see >> (2 * i) & 1u ? x : -INFINITY, y = see >> (2 * i + 1) & 1u ? y : -INFINITY;
                            }
                            const uint64_t p2 = f2pack(ex2(x), ex2(y));
                            sum2 = fadd2(sum2, p2);
                            f2unpack(p2, x, y);
                            if (PARTS == 1) {
                                hi[i] = ts_pack<BF16>(x, y);
                            } else {
                                // the remainder is above 0, so that its product with an infinite value has the sign of
                                // the other part's (2^-38 of the row's largest weight is far below F32's last bit)
                                hi[i] = ts_pack_rz<BF16>(x, y);
                                const float2 f = ts_unpack<BF16>(hi[i]);
                                f2unpack(ffma2(f2pack(f.x, f.y), f2pack(-1.0f, -1.0f), p2), x, y);
                                lo[i] = masked ? ts_pack<BF16>(x, y) : ts_positive<BF16>(ts_pack<BF16>(x, y));
                            }
                        }
                        tmem_st16(s_col + (uint32_t) (c * 16 * PARTS), hi);
                        if (PARTS == 2) {
                            tmem_st16(s_col + (uint32_t) (c * 32 + 16), lo);
                        }
                    }
                    float x, y;
                    f2unpack(sum2, x, y);
                    l = fmaf(l, g, x + y);
                    tmem_st_wait();
                }
                tc_fence_before();
                dn_mbar_arrive(&bar[TB_PREADY + w]);
                wait(TB_OFULL + w, tc >> 1);
                if (warp_live) {
#pragma unroll
                    for (int c = 0; c < D / 32; c++) {
                        uint32_t o[32];
                        tmem_ld32(o_col + (uint32_t) (c * 32), o);
                        tmem_ld_wait_tie(o);
#pragma unroll
                        for (int e = 0; e < 32; e++) {
                            acc[c * 32 + e] = fmaf(acc[c * 32 + e], g, __uint_as_float(o[e]));
                        }
                    }
                }
                tc_fence_before();
                dn_mbar_arrive(&bar[TB_OFREE + w]);
            }
            // ---- the two streams' maxima and sums, then each takes half of the columns
            ml[w * TS_M + r] = make_float2(m, l);
            softmax_barrier();
            const float2 other = ml[(w ^ 1) * TS_M + r];
            const float  M = fmaxf(m, other.x), mine_f = m == M ? 1.0f : ex2(m - M), other_f = other.x == M ? 1.0f : ex2(other.x - M);
            l = w == 0 ? fmaf(l, mine_f, other.y * other_f) : fmaf(other.y, other_f, l * mine_f);
            l = f0 != f0 && M != -INFINITY ? NAN : l;
            float res[D / 2];
#pragma unroll
            for (int c = 0; c < D / 64; c++) {
                // to the other stream: columns 32 c .. of its half
                float4 * give = xch + w * (TS_M * 8), *take = xch + (w ^ 1) * (TS_M * 8);
#pragma unroll
                for (int k = 0; k < 8; k++) {
                    float4 f;
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        (&f.x)[e] = w ? acc[c * 32 + k * 4 + e] : acc[D / 2 + c * 32 + k * 4 + e];
                    }
                    give[r * 8 + (k ^ (r & 7))] = f;
                }
                softmax_barrier();
#pragma unroll
                for (int k = 0; k < 8; k++) {
                    const float4 f = take[r * 8 + (k ^ (r & 7))];
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        const float a = w ? acc[D / 2 + c * 32 + k * 4 + e] : acc[c * 32 + k * 4 + e];
                        // (the same operations in the same order whichever stream's it is)
                        res[c * 32 + k * 4 + e] = a * mine_f + (&f.x)[e] * other_f;
                    }
                }
                softmax_barrier();
            }
            const int at = w * (D / 2);  // this thread's columns
            if (tail && *dirty && live) {
                // elements that are no numbers, of nodes that the row sees: they were left out of the products
                for (int n = 0; n < nodes; n++) {
                    const int key = held + n;
                    if (key / TS_N < it.a || key / TS_N >= it.b || !(bits[n >> 5] >> (n & 31) & 1u)) {
                        continue;
                    }
                    const uint16_t * v = reinterpret_cast<const uint16_t *>(p.v.data + (int64_t) key * p.v.nb1 + (int64_t) it.h * p.v.nb2 + (int64_t) it.s * p.v.nb3) + at;
#pragma unroll
                    for (int e = 0; e < D / 2; e++) {
                        const float x = ts_unpack<BF16>(v[e]).x;
                        res[e] += fabsf(x) < INFINITY ? 0.0f : x;
                    }
                }
            }
            // ---- the result, or a part's sums into the workspace
            {
                const bool whole = it.a == 0 && it.b == it.q.tiles;
                uint64_t   al;  // where this row goes
                if (whole) {
                    const int hd = it.h * p.ratio + row - my_node * p.ratio;
                    al = reinterpret_cast<uint64_t>(p.o.data + (int64_t) hd * p.o.nb1 + (int64_t) my_node * p.o.nb2 + (int64_t) it.s * p.o.nb3);
                } else {
                    // the unit's parts: the first belongs to the piece before the first one that starts inside the unit, in its
                    // second slot unless the unit is its first; the others are their pieces' first
                    const int     pa = it.a == 0 ? group + 1 : ln.last(it.unit + TS_LEAST - 1) + 1, floats = ts_slot_floats(slot_rows, D);
                    const int64_t step = (int64_t) blocks * 2 * floats, part1 = ((int64_t) pa * blocks + rb) * 2 * floats;
                    const int64_t part0 = part1 - step + (ln.at(pa - 1) <= it.unit - TS_LEAST ? floats : 0);
                    float *       slot  = p.part + (it.a == 0 ? part0 : part1 + (group - pa) * step);
                    al = reinterpret_cast<uint64_t>(slot + r * D);
                    if (live && w == 0) {
                        *reinterpret_cast<float2 *>(slot + slot_rows * D + 2 * r) = make_float2(M, l);
                    }
                    if (own == 0 && it.a == 0) {
                        *join = { it.s, it.h, ln.last(it.unit + it.q.tiles - TS_LEAST) - pa + 2, its_rows, part0, part1 };
                    }
                }
                // by whole rows, 32 columns at a time through this warp's part of the exchange
                const float inv   = whole ? (l != 0.0f ? 1.0f / l : 0.0f) : 1.0f;
                float4 *    stage = xch + w * (TS_M * 8) + quad * 32 * 8;
                const int   type = whole ? p.o.type : (int) KV_F32;
                const bool  vec = !whole || p.o.vec;
                if (warp_live) {
#pragma unroll
                    for (int c = 0; c < D / 64; c++) {
#pragma unroll
                        for (int k = 0; k < 8; k++) {
                            stage[lane * 8 + (k ^ (lane & 7))] = make_float4(res[c * 32 + k * 4] * inv, res[c * 32 + k * 4 + 1] * inv,
                                                                             res[c * 32 + k * 4 + 2] * inv, res[c * 32 + k * 4 + 3] * inv);
                        }
                        __syncwarp();
#pragma unroll 1
                        for (int i = lane >> 3; i < 32; i += 4) {
                            const int    k = lane & 7;
                            const float4 f = stage[i * 8 + (k ^ (i & 7))];
                            char *       to = reinterpret_cast<char *>(__shfl_sync(0xffffffffu, al, i));
                            if (quad * 32 + i < its_rows) {
                                ts_store4(to, at + c * 32 + k * 4, f, type, vec);
                            }
                        }
                        __syncwarp();
                    }
                }
            }
            softmax_barrier();  // Q's memory and the ancestors are free
            if (own == 0) {
                *dirty = 0;  // (the next piece's tiles are looked at when all threads have staged its Q)
            }
        }
        if (!ok) {
            atomicExch(abort_f, 1);
        }
    }

    tc_fence_before();
    __syncthreads();
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc(tmem, TS_TMEM);
    }
    if (tid == 0 && *abort_f) {
        kv8_report(p.status, ST_TIMEOUT);
        atomicExch(&p.status[1], blockIdx.x);
    }
}

// Joins the parts of units: one row by D / 4 lanes, the parts in their order.
template <int D>
__global__ void __launch_bounds__(TJ_ROWS * D / 4) tree_attn_join_kernel(const TreeAttnParams p, int blocks, int slot_rows) {
    kv8_dep_wait();
    constexpr int PER = 8;  // parts loaded at a time
    const TsJoin  t   = *(reinterpret_cast<const TsJoin *>(reinterpret_cast<const char *>(p.status) + TS_SPACE) + blockIdx.x);
    const int     rb = (int) blockIdx.x % blocks, lane = threadIdx.x % (D / 4), r = (int) blockIdx.y * TJ_ROWS + threadIdx.x / (D / 4);
    if (t.parts == 0 || r >= t.rows) {
        return;
    }
    const int64_t step = (int64_t) blocks * 2 * ts_slot_floats(slot_rows, D);
    auto          part = [&](int k) { return p.part + (k == 0 ? t.part0 : t.part1 + (k - 1) * step); };
    float         M = -INFINITY, l = 0.0f;
    float4        o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    for (int k0 = 0; k0 < t.parts; k0 += PER) {
        float2 x[PER];
        float4 v[PER];
#pragma unroll
        for (int k = 0; k < PER; k++) {
            const float * at = part(min(k0 + k, t.parts - 1));
            x[k] = *reinterpret_cast<const float2 *>(at + slot_rows * D + 2 * r);
            v[k] = *(reinterpret_cast<const float4 *>(at + r * D) + lane);
        }
        float top = M;
#pragma unroll
        for (int k = 0; k < PER; k++) {
            top = fmaxf(top, x[k].x);
        }
        const float g = M == top ? 1.0f : ex2(M - top);
        l *= g, o.x *= g, o.y *= g, o.z *= g, o.w *= g, M = top;
#pragma unroll
        for (int k = 0; k < PER; k++) {
            if (k0 + k < t.parts) {
                const float f = x[k].x == M ? 1.0f : ex2(x[k].x - M);
                l = fmaf(x[k].y, f, l);
                o.x = fmaf(v[k].x, f, o.x), o.y = fmaf(v[k].y, f, o.y), o.z = fmaf(v[k].z, f, o.z), o.w = fmaf(v[k].w, f, o.w);
            }
        }
    }
    const float inv = l != 0.0f ? 1.0f / l : 0.0f;
    const int   row = rb * TS_M + r, node = row / p.ratio, head = t.h * p.ratio + row - node * p.ratio;
    ts_store4(p.o.data + (int64_t) head * p.o.nb1 + (int64_t) node * p.o.nb2 + (int64_t) t.s * p.o.nb3, 4 * lane,
              make_float4(o.x * inv, o.y * inv, o.z * inv, o.w * inv), p.o.type, p.o.vec);
}

template <int D, bool BF16, int PARTS>
cudaError_t launch_one(const TreeAttnParams & p, int sms, cudaStream_t stream) {
    auto             kern = tree_attn_tc_kernel<D, BF16, PARTS>;
    static Kv8Once   once;
    static const int regs = [&] {
        cudaFuncAttributes a{};
        return cudaFuncGetAttributes(&a, kern) == cudaSuccess ? a.numRegs : 0;
    }();
    // the register split draws on what the launch gives: another count would wait for registers that never come
    if (regs != TS_REGS_LAUNCH) {
        return cudaErrorInvalidConfiguration;
    }
    constexpr int smem = TsSmem<D, PARTS>::TOTAL;
    cudaError_t   e    = once.smem(kern, smem);
    if (e != cudaSuccess) {
        return e;
    }
    alignas(64) CUtensorMap tmk, tmv;
    if (!encode_kv_tensor_map(&tmk, p.k.data, BF16, D, p.n_kv, p.n_head_kv, p.n_seq, p.k.nb1, p.k.nb2, p.k.nb3, TS_N) ||
        !encode_kv_tensor_map(&tmv, p.v.data, BF16, D, p.n_kv, p.n_head_kv, p.n_seq, p.v.nb1, p.v.nb2, p.v.nb3, TS_N)) {
        return cudaErrorInvalidValue;
    }
    const int blocks = tree_attn_blocks(p), groups = tree_attn_groups(p, sms);
    const int rows = std::min(p.t.max_nodes * p.ratio, TS_M);
    e = kv8_launch(kern, dim3((unsigned) (groups * blocks)), TS_THREADS, smem, stream, tmk, tmv, p, blocks, groups, rows);
    if (e != cudaSuccess || p.n_kv <= (2 * TS_LEAST - 1) * TS_N) {
        return e;  // (no unit is in parts)
    }
    return kv8_launch(tree_attn_join_kernel<D>, dim3((unsigned) (groups * blocks), (unsigned) ((rows + TJ_ROWS - 1) / TJ_ROWS)), TJ_ROWS * D / 4, 0, stream, p,
                      blocks, rows);
}

template <int D, bool BF16>
cudaError_t launch_d(const TreeAttnParams & p, int sms, cudaStream_t stream) {
    // one part where q is the cache's type and the result has no more bits
    return p.q.type == p.k.type && p.o.type == p.q.type ? launch_one<D, BF16, 1>(p, sms, stream) : launch_one<D, BF16, 2>(p, sms, stream);
}

}  // namespace

// 16-bit slabs whose strides a tensor map takes, at D = 64 and 128
bool tree_attn_tc_takes(const TreeAttnParams & p) {
    for (const Kv8Rows * x : { &p.k, &p.v }) {
        const int64_t most = (int64_t) 1 << 40;
        if (!x->vec || (p.n_kv > 1 && (x->nb1 < 2 * p.D || x->nb1 >= most)) || (p.n_head_kv > 1 && (x->nb2 <= 0 || x->nb2 >= most)) ||
            (p.n_seq > 1 && (x->nb3 <= 0 || x->nb3 >= most))) {
            return false;
        }
    }
    return (p.k.type == KV_F16 || p.k.type == KV_BF16) && (p.D == 64 || p.D == 128) && tensor_maps_available() &&
           (int64_t) p.n_seq * p.n_head_kv * ((p.n_kv + TS_N - 1) / TS_N) < (1 << 30);
}

int tree_attn_blocks(const TreeAttnParams & p) {
    return (p.t.max_nodes * p.ratio + TS_M - 1) / TS_M;
}

int tree_attn_groups(const TreeAttnParams & p, int sms) {
    const int64_t tiles = (int64_t) p.n_seq * p.n_head_kv * ((p.n_kv + TS_N - 1) / TS_N);
    return (int) std::max<int64_t>(1, std::min<int64_t>(sms / tree_attn_blocks(p), tiles));
}

size_t tree_attn_tc_workspace(const TreeAttnParams & p, int sms) {
    const int blocks = tree_attn_blocks(p), rows = std::min(p.t.max_nodes * p.ratio, TS_M);
    return KV8_WS_ZEROED + (size_t) tree_attn_groups(p, sms) * blocks * 2 * ts_slot_floats(rows, p.D) * 4;
}

cudaError_t launch_tree_attn_tc(TreeAttnParams p, int sms, cudaStream_t stream) {
    p.part     = reinterpret_cast<float *>(reinterpret_cast<char *>(p.status) + KV8_WS_ZEROED);
    if (p.D == 64) {
        return p.k.type == KV_BF16 ? launch_d<64, true>(p, sms, stream) : launch_d<64, false>(p, sms, stream);
    }
    return p.k.type == KV_BF16 ? launch_d<128, true>(p, sms, stream) : launch_d<128, false>(p, sms, stream);
}

}  // namespace mm3fa
