// tree_attn_sm100.cu - attention of a tree of drafted tokens over a 16-bit slab cache on the 5th-generation tensor cores
// (tcgen05 + TMEM), sm_100a.
//
// Rows of a unit (sequence, kv head) are (node, head of the group) pairs in that order; a block has 128 of them, so the
// query heads of a kv head and the nodes share each K/V tile of 128 keys.  One CTA per SM.  Where all trees have the same
// nodes, the CTAs with a unit's blocks are a group, beside one another, that walks the same keys at the same time, so that
// a K/V tile comes from HBM once; where each tree says how many it has, the blocks are units of their own, since a group's CTAs
// would have nothing to do for the smaller trees (8 trees of up to 200 nodes, before later steps: 128 us in groups of 7, 99 as
// units).
//
// Split, found on the device from the lengths, so that a captured call follows them:
//   units up to groups   every unit in even parts of about the same size, one part a group (TsPlan; 2 sequences of 8192: 30 us,
//                        37 on a line; of 97 and 311: 17 and 32)
//   more units           the tiles of all units are one line, in the order of sequence and kv head, and each group takes an
//                        equal piece of it: whole units, and a part of one at either end
// A part of a unit leaves O, m and l in the workspace, and a second kernel joins the parts in their order: by the last
// CTA to arrive, one SM of 148 would read all parts of a unit (25 us for 9 parts of 96 rows, at one SM's bandwidth).
// That kernel is left out where the slab is too short for a part.
//
// 384 threads:
//   warp 0       TMA: K and V tiles through one ring, in the order in which the products take them
//   warp 1       TMEM allocation and every tcgen05.mma: QK(j + 1), then P V(j), P in TMEM over S (a third part behind it)
//   warps 2, 3   the V rows of tiles that hold nodes: those behind the last node become zero, and so do elements that are
//                no numbers (their weight may be 0; who sees such a node gets them added at the end); then the next
//                piece's Q, beside the softmax of this one's last tiles
//   warpgroups 1, 2   softmax of the even and the odd tiles, one row per thread: two streams with maxima, sums and O of their
//                own, joined at the piece's end
//
// Numerics.  Where q has the cache's type and the result no more bits (PARTS 1), O stays in TMEM and is multiplied there when
// a row's maximum grows by more than 2^TS_GROW.  The tensor core truncates what it adds to an accumulator, up to 2^-23 of it in
// each step of 16 keys, always towards zero (measured 7e-7 a tile of 128 keys): up to TS_LONG keys a stream's sum stays within
// 1e-4, a fifth of F16's half step.  Else (PARTS 2) q is two parts of the cache's type (brought to [2^14, 2^15), BF16 to [1, 2), at
// its row's largest element by a power of two), and so are the weights, the remainder's product first, where the accumulator is small;
// every tile's P V starts afresh and is added in registers, rounded to nearest: 22 bits of q and weights in F16 (an F32 result
// is off by 5e-7 of its norm), 16 in BF16, which F32 results over BF16 slabs take three parts for (PARTS 3: 24 bits; 4e-7 of the
// norm, 3.5e-6 with two), in tiles of 64 keys, as TMEM has no place for three parts of 128.  2 x 8192, 24 nodes: PARTS 1 22 us
// (BF16), 2 31, 3 39; 64 nodes: 32, 49, 68; 48 sequences of up to 10240, 13 nodes: 166, 249, 355 (tiles of 80 keys, the most that
// TMEM takes, were no faster).
//
// Bound: HBM for batches at full clock (48 sequences of 1 to 10240, 13 nodes, BF16, 1013 MB: 166 us, 6.1 TB/s, at 1965 MHz; under a
// lasting load the power cap takes the clock to 1430-1550 MHz, and the tiles' own work counts too: 177-188); few sequences
// the start (plan 2.7 us, Q 6, first S 7.6) and the joining (7); many nodes each stream's chain of S, weights, P V (2 us a tile, the tensor pipe 38%
// active), and the ends of pieces (8 trees of up to 200 nodes over 1900-4100 tokens: 80 us for 45.6 GFLOP).
//
// Most of the code runs once in a CTA, and its first run costs what the instruction cache costs: what does not feed the
// tensor core is in rolled loops or functions (a Q staging unrolled over all rows took 5 us, 3.5 as it is).
#include "fa_decode.cuh"
#include "tc_sm100.cuh"
#include "tree.cuh"

#include <algorithm>

namespace mm3fa {

namespace {

constexpr int TS_THREADS = 384;
constexpr int TS_M       = 128;  // rows of a block
constexpr int TS_S       = 128;  // columns of a tile's S, with the weights over it
constexpr int TS_TMEM    = 512;  // columns: S of two tiles, P V of two tiles
constexpr int TS_GROW    = 7;    // (PARTS 1) log2 of what a weight may exceed the maximum of the tiles before by
constexpr int TS_LONG    = 32768;
constexpr int TS_SPACE   = 256;  // bytes of the workspace before the list of units in parts
constexpr int TS_LEAST   = 3;    // tiles of a part, at least (8 trees of up to 200 nodes: 79 us, 82 with 4, 85 with 8)
constexpr int TS_PIECES  = 4;    // pieces that warp 0 may be ahead
constexpr int TS_COST    = 5;    // tiles' time that a unit takes beside them
constexpr int TS_EVEN    = 160;  // sequences for which even parts are looked for: five for each lane
constexpr int TJ_WARPS   = 8;    // of a joining CTA
constexpr int TJ_UNITS   = 512;  // units in parts, at most one a CTA: there are no more CTAs than SMs or blocks of a unit
constexpr float TS_MOST       = 3.402823466e38f;  // F32's largest number
constexpr int TS_REGS_LAUNCH  = 168;  // 65536 / 384, a multiple of 8
constexpr int TS_REGS_SOFTMAX = 208;  // 2 x 208 + 88 = 3 x 168
constexpr int TS_REGS_ISSUE   = 88;
static_assert(2 * TS_REGS_SOFTMAX + TS_REGS_ISSUE <= 3 * TS_REGS_LAUNCH, "more registers than the launch has");

// log2 of what a weight at the maximum is held as: F16 keeps 11 bits of one down to 2^-(14 + offset) of it, and holds 2^15;
// BF16, whose small numbers go as far as F32's, holds none above 1, so that sums of large values stay in F32
template <bool BF16, int PARTS>
constexpr float TS_OFF = BF16 ? (PARTS >= 2 ? 0.0f : -(float) TS_GROW) : PARTS >= 2 ? 14.0f : 15.0f - TS_GROW;

// keys of a tile: three parts of the weights of 128 keys would have no place in TMEM
__host__ __device__ constexpr int ts_keys(int parts) {
    return parts == 3 ? 64 : 128;
}

template <int D, int PARTS>
struct TsSmem {
    static constexpr int N      = ts_keys(PARTS);
    static constexpr int HALVES = D / 64;  // 128-byte column blocks
    static constexpr int QT     = HALVES * TS_M * 128;
    static constexpr int KT     = HALVES * N * 128;
    static constexpr int NS     = D == 128 ? (PARTS == 3 ? 6 : PARTS == 2 ? 4 : 5) : 8;  // tiles in the ring
    static constexpr int OFF_Q    = 0;
    static constexpr int OFF_RING = OFF_Q + PARTS * QT;
    static constexpr int OFF_XCH  = OFF_RING + NS * KT;           // [stream][row] 16 columns
    static constexpr int OFF_ANC  = OFF_XCH + 2 * TS_M * 64;      // [TREE_MAX][TREE_MAX / 32] bits
    static constexpr int OFF_PAR  = OFF_ANC + TREE_MAX * (TREE_MAX / 32) * 4;
    static constexpr int OFF_F    = OFF_PAR + TREE_MAX * 4;       // [2 pieces][row] factors
    static constexpr int OFF_ML   = OFF_F + 2 * TS_M * 4;         // [stream][row] (m, l)
    static constexpr int OFF_BAR  = OFF_ML + 2 * TS_M * 8;
    static constexpr int OFF_PIECE = OFF_BAR + 40 * 8;            // [TS_PIECES]
    static constexpr int OFF_MISC  = OFF_PIECE + TS_PIECES * 64;
    static constexpr int TOTAL     = OFF_MISC + 32 + 1024;        // + alignment
};
static_assert(TsSmem<128, 1>::TOTAL <= 232448 && TsSmem<128, 2>::TOTAL <= 232448 && TsSmem<128, 3>::TOTAL <= 232448 && TsSmem<64, 2>::TOTAL <= 232448, "shared memory");

enum : int {
    TB_FULL   = 0,   // [8] TMA
    TB_EMPTY  = 8,   // [8] products
    TB_SFULL  = 16,  // [2]
    TB_PREADY = 18,  // [2] 128 softmax threads
    TB_OFULL  = 20,  // [2] a tile's P V (PARTS 1: the last of a piece)
    TB_QREADY = 22,  // [2 pieces] 64.  (Two: a piece's may follow the one before while the softmax has not waited for that yet)
    TB_QFREE  = 24,  // the last QK of a piece
    TB_LOOK   = 25,  // warp 1: a V tile with nodes is there
    TB_FIX    = 26,  // 64 threads of warps 2, 3: it can be taken
    TB_DONE   = 27,
    TB_PIECE  = 28,  // [TS_PIECES] warp 0
    TB_PFREE  = 32,  // [TS_PIECES] the 11 other warps
    TB_COUNT  = 36,
};

__host__ __device__ constexpr uint32_t ts_arrivals(int b) {
    return b >= TB_PFREE ? (uint32_t) (TS_THREADS / 32 - 1) : b == TB_QREADY || b == TB_QREADY + 1 || b == TB_FIX ? 64u : b == TB_PREADY || b == TB_PREADY + 1 ? 128u : 1u;
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

__device__ __forceinline__ void tmem_st8(uint32_t taddr, const uint32_t * r) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]),
                 "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
                 : "memory");
}

__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t * r) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]),
          "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(taddr)
        : "memory");
}

__device__ __forceinline__ void tmem_ld16_wait(uint32_t * r) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]), "+r"(r[9]), "+r"(r[10]),
                   "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15])
                 :
                 : "memory");
}

__device__ __forceinline__ void softmax_barrier() {  // the 256 threads of both streams
    asm volatile("bar.sync 1, 256;" ::: "memory");
}

__device__ __forceinline__ bool softmax_all(bool x) {  // the same, and whether x holds for all of them
    uint32_t all;
    asm volatile(
        "{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %1, 0;\n\t"
        "barrier.cta.red.and.pred q, 1, 256, p;\n\tselp.u32 %0, 1, 0, q;\n\t}"
        : "=r"(all)
        : "r"(x ? 1u : 0u)
        : "memory");
    return all != 0;
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

template <bool BF16>
__device__ __forceinline__ float2 ts_unpack(uint32_t u) {
    return BF16 ? bf2_to_f2(u) : h2_to_f2(u);
}

// tanh within 4e-7 of its value: (1 - e) / (1 + e) with e = exp(-2 |x|), below 1/4 its series (a call would not leave the
// registers that the softmax has)
__device__ __forceinline__ float ts_tanh(float x) {
    const float a = fabsf(x), e = ex2(-2.0f * LOG2E * a), x2 = x * x;
    const float t = __fdividef(1.0f - e, 1.0f + e), p = fmaf(fmaf(fmaf(-17.0f / 315.0f, x2, 2.0f / 15.0f), x2, -1.0f / 3.0f) * x2, a, a);
    return copysignf(a < 0.25f ? p : t, x);
}

// Floats of a part: O as [D / 4][row] of four, then m and l of each row; a multiple of 16 bytes.
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
    int     s, h, parts, rows;  // parts 0: the CTA has no such unit
    int64_t row0;               // the block's first row
    int64_t part0, part1;       // where the first part and the second are, in floats; the others follow at even steps
};

// a / b for 0 <= a and 0 < b.  Below 2^20 in F32: (a + 1/2) / b is at least 1 / 2b from a whole number, and off by less.
__device__ __noinline__ int ts_div_large(int a, int b) {
    return (int) ((unsigned) a / (unsigned) b);
}

__device__ __forceinline__ int ts_div(int a, int b) {
    return a < (1 << 20) ? (int) __fdividef((float) a + 0.5f, (float) b) : ts_div_large(a, b);
}

__device__ __forceinline__ int ts_up(int a, int b) {
    return ts_div(a + b - 1, b);
}

// Key tiles of a sequence's units; 0 where none of its nodes counts.
struct TsSeq {
    int L, nodes, keys, tiles;
};

template <int N>
__device__ __forceinline__ TsSeq ts_seq(const TreeAttnParams & p, int s) {
    TsSeq q;
    q.nodes = tree_nodes(p.t, s % p.t.n_tree);
    q.L     = min(max(p.kv_len[s], 0), p.n_kv);
    q.keys  = q.nodes > 0 ? min(q.L + q.nodes, p.n_kv) : 0;
    q.tiles = (q.keys + N - 1) / N;
    return q;
}

// The line of all units' tiles, each unit with TS_COST more, in G even pieces, piece g from `at(g)` on.  A border closer than
// TS_LEAST tiles to a unit's start or end goes there, so that no part of a unit has less.
struct TsLine {
    int W, G, each, more;  // `more` pieces have a tile more than `each`

    __device__ __forceinline__ void cut(int W_, int groups) {
        W    = W_;
        G    = max(1, min(groups, W_ / (TS_COST + TS_LEAST)));
        each = ts_div(W, G);
        more = W - each * G;
    }

    __device__ __forceinline__ int at(int g) const {
        return g * each + min(g, more);
    }

    // the last piece that starts at tile x or before
    __device__ __forceinline__ int last(int x) const {
        const int y = more * (each + 1);
        return min(G - 1, x < y ? ts_div(x, each + 1) : each > 0 ? more + ts_div(x - y, each) : G - 1);
    }

    // border x, of a unit that starts at `first`, is n long and holds x
    static __device__ __forceinline__ int border(int x, int first, int n) {
        return x - first < TS_COST + TS_LEAST ? first : first + n - x < TS_LEAST ? first + n : x;
    }
};

// Tiles [a, b) of a unit, for one block of its rows, as warp 0 tells the others.
struct __align__(16) TsPiece {
    int     s, h, a, b;
    int     rb, rows;               // the block of rows, how many it has; 0: there is no further piece
    int     L, nodes, keys, tiles;  // of the sequence
    int     unit;                   // where the unit starts
    int64_t slot;                   // floats, where it is a part
};

static_assert(sizeof(TsPiece) == 64, "shared memory");

// A group's pieces, one after another.
template <int N>
struct TsPlan {
    const TreeAttnParams & p;
    int                    group, beside, wide, floats;  // floats of a part's slot; a CTA has two
    int                    even;                         // 0, or the tiles of a part, at most
    TsLine                 ln;
    int                    s, first, x, end;  // first: of sequence s on the line (even: among the parts); end: before its move to a border
    TsSeq                  q;

    // wide: the CTAs of a group, each with the block of its place (1: the blocks are units of their own)
    __device__ __forceinline__ TsPlan(const TreeAttnParams & p_, int wide_, int floats_)
        : p(p_), group((int) blockIdx.x / wide_), beside((int) blockIdx.x % wide_), wide(wide_), floats(floats_), even(0), s(0), first(0), x(0), end(0), q{ 0, 0, 0, 0 } {}

    __device__ __forceinline__ void find(int groups) {  // by a whole warp
        // each lane sums some sequences; all tiles are fewer than 2^30 (checked by the host)
        const int lane = threadIdx.x & 31, each = (p.n_seq + 31) / 32, s0 = min(lane * each, p.n_seq), s1 = min(s0 + each, p.n_seq);
        int       mine = 0, units = 0, most = 0;
        TsSeq     own = { 0, 0, 0, 0 };  // the lane's last sequence, its only one where there are up to 32
#pragma unroll 1
        for (int i = s0; i < s1; i++) {
            own = ts_seq<N>(p, i);
            mine += own.tiles * heads(own), units += own.tiles > 0 ? heads(own) : 0, most = max(most, own.tiles);
        }
        const int W = __reduce_add_sync(0xffffffffu, mine), U = __reduce_add_sync(0xffffffffu, units);
        most = __reduce_max_sync(0xffffffffu, most);
        int from, to;
        if (p.n_seq <= TS_EVEN && U <= groups) {
            // the fewest tiles to a part that need no more than all groups: each lane tries one of 32 numbers between what
            // even shares would be and what is enough
            const int lo = max(TS_LEAST + 1, ts_up(W + U, groups));
            const int hi = max(lo, U < groups ? min(most + 1, ts_up(W + U, groups - U)) : most + 1);
            const int t  = lo + lane * ((hi - lo + 30) / 31);
            int       parts = 0;
#pragma unroll 1
            for (int i = 0; i < p.n_seq; i++) {
                TsSeq c = own;
                if (each == 1) {
                    c.tiles = __shfl_sync(0xffffffffu, own.tiles, i), c.nodes = __shfl_sync(0xffffffffu, own.nodes, i);
                } else {
                    c = ts_seq<N>(p, i);
                }
                parts += c.tiles > 0 ? ts_up(c.tiles + 1, t) * heads(c) : 0;
            }
            const unsigned fits = __ballot_sync(0xffffffffu, parts <= groups);
            even = __shfl_sync(0xffffffffu, t, __ffs(fits) - 1);  // (the last lane's fits)
            mine = 0;
#pragma unroll 1
            for (int i = s0; i < s1; i++) {
                mine += weight(each == 1 ? own : ts_seq<N>(p, i));
            }
            from = group, to = group + 1;
        } else {
            ln.cut(W + U * TS_COST, groups);
            from = group < ln.G ? ln.at(group) : ln.W, to = group < ln.G ? ln.at(group + 1) : ln.W;
            mine += units * TS_COST;
        }
        int at = mine;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const int y = __shfl_up_sync(0xffffffffu, at, d);
            at += lane >= d ? y : 0;
        }
        at -= mine;
        const unsigned here = __ballot_sync(0xffffffffu, from < to && from >= at && from < at + mine);  // it starts among this lane's
        if (here == 0) {
            return;  // (nothing for this group)
        }
        int i = s0;
        if (each > 1 && (here >> lane & 1u)) {
#pragma unroll 1
            for (;; i++) {
                const int n = weight(ts_seq<N>(p, i));
                if (from < at + n) {
                    break;
                }
                at += n;
            }
        }
        const int src = __ffs(here) - 1;
        s = __shfl_sync(0xffffffffu, i, src), first = __shfl_sync(0xffffffffu, at, src);
        q = each == 1 ? TsSeq{ __shfl_sync(0xffffffffu, own.L, src), __shfl_sync(0xffffffffu, own.nodes, src), __shfl_sync(0xffffffffu, own.keys, src),
                               __shfl_sync(0xffffffffu, own.tiles, src) } :
                        ts_seq<N>(p, s);
        x = from, end = to;
        if (!even) {
            x = TsLine::border(x, first + ts_div(x - first, q.tiles + TS_COST) * (q.tiles + TS_COST), q.tiles + TS_COST);
        }
    }

    // units of a sequence: its kv heads, by its blocks of rows where these are on their own
    __device__ __forceinline__ int heads(const TsSeq & c) const {
        return wide > 1 ? p.n_head_kv : p.n_head_kv * ((c.nodes * p.ratio + TS_M - 1) / TS_M);
    }

    // a unit's length on the line, or its parts: these share its tiles and one more, for what the nodes' masks take
    __device__ __forceinline__ int length(const TsSeq & c) const {
        return even ? ts_up(c.tiles + 1, even) : c.tiles + TS_COST;
    }

    // a sequence's
    __device__ __forceinline__ int weight(const TsSeq & c) const {
        return c.tiles == 0 ? 0 : length(c) * heads(c);
    }

    // the next piece that has rows in this CTA's block
    __device__ __forceinline__ TsPiece next() {
        TsPiece c = {};
#pragma unroll 1
        while (x < end) {
            const int n = q.tiles > 0 ? length(q) : 0, all = n * heads(q);
            if (x - first >= all) {
                first += all;
                q = ts_seq<N>(p, ++s);
                continue;
            }
            const int i = ts_div(x - first, n);  // the unit
            const int bl = wide > 1 ? 1 : (q.nodes * p.ratio + TS_M - 1) / TS_M;
            c.h    = bl == 1 ? i : ts_div(i, bl);
            c.rb   = wide > 1 ? beside : i - c.h * bl;
            c.rows = min(q.nodes * p.ratio - c.rb * TS_M, TS_M);
            if (c.rows <= 0) {  // (the block is empty: on to the next sequence)
                c.rows = 0;
                x      = first + all;
                continue;
            }
            c.s = s, c.L = q.L, c.nodes = q.nodes, c.keys = q.keys, c.tiles = q.tiles;
            c.unit = first + i * n;
            if (even) {
                const int k = x - c.unit;
                c.a = ts_div(k * (q.tiles + 1), n), c.b = min(ts_div((k + 1) * (q.tiles + 1), n), q.tiles);
                x++;
            } else {
                const int to = c.unit + n <= end ? c.unit + n : TsLine::border(end, c.unit, n);
                c.a = max(x - c.unit - TS_COST, 0), c.b = to - c.unit - TS_COST;
                if (to <= x) {
                    c.rows = 0;
                }
                x = c.rows ? to : end;
            }
            c.slot = part(c, second(c), group - second(c) + 1);
            return c;
        }
        c.rows = 0;
        return c;
    }

    // the group that has the second part of a piece's unit
    __device__ __forceinline__ int second(const TsPiece & c) const {
        return even ? c.unit + 1 : c.a == 0 ? group + 1 : ln.last(c.unit + TS_COST + TS_LEAST - 1) + 1;
    }

    // Where a unit's parts are: the first in a slot of the group before `g`, its second one unless the unit is the first that
    // the group has; the others in the first slots of g and the groups behind it.
    __device__ __forceinline__ int64_t part(const TsPiece & c, int g, int k) const {
        const int64_t slots = ((int64_t) (g - 1 + k) * wide + beside) * 2;
        return (slots + (k == 0 && !even && ln.at(g - 1) <= c.unit - TS_LEAST ? 1 : 0)) * floats;
    }

    // what the joining kernel has to know of a unit, from its first part
    __device__ __forceinline__ TsJoin join(const TsPiece & c) const {
        const int g = second(c), parts = even ? ts_up(c.tiles + 1, even) : ln.last(c.unit + c.tiles + TS_COST - TS_LEAST) - g + 2;
        return { c.s, c.h, parts, c.rows, c.rb * TS_M, part(c, g, 0), part(c, g, 1) };
    }
};

// Rows ra .. ra + 15 of a block's Q for the products, by a warp; rows that do not count are zeros.  All copies are in
// flight at once, and land where the row's products will read it: PARTS 1, as they are; else a row's bytes lie in the
// places of its own first two parts (F32: all of them), and the warp replaces one row after another.
template <int D, bool BF16, int PARTS, int UNROLL>
__device__ __forceinline__ void ts_stage16(const TreeAttnParams & p, const TsPiece & it, int ra, char * qs, float * factors, int lane) {
    constexpr int E = D / 32, QT = TsSmem<D, PARTS>::QT, BLOCK = TS_M * 128;
    const int     in = it.rows - ra, esz = p.q.type == KV_F32 ? 4 : 2;
    // lane i, and 16 + i: the address of row i (of the last one, behind it)
    const int      rl = it.rb * TS_M + max(min(ra + (lane & 15), it.rows - 1), 0), nl = rl / p.ratio, hl = it.h * p.ratio + rl - nl * p.ratio;
    const uint64_t al = reinterpret_cast<uint64_t>(p.q.data + (int64_t) nl * p.q.nb1 + (int64_t) hl * p.q.nb2 + (int64_t) it.s * p.q.nb3);
    const float    by = fabsf(p.softcap > 0.0f ? p.scale / p.softcap : p.scale * LOG2E);
    // chunk ck of 16 bytes of row i: block ck / 8 of 64 columns (F32: the two blocks of either part in turn)
    auto place = [&](int i, int ck) {
        const int blk = ck >> 3;
        return qs + (blk % (D / 64)) * BLOCK + (blk / (D / 64)) * QT + (ra + i) * 128 + (((ck & 7) ^ (PARTS == 1 ? i & 7 : 0)) << 4);  // (ra: a multiple of 8)
    };
    const int chunks = D * esz / 16, per = 32 / chunks, ck = lane % chunks, i1 = lane / chunks;
    if (p.q.vec) {
#pragma unroll UNROLL
        for (int i = i1; i < 16; i += per) {
            const uint64_t src = __shfl_sync(0xffffffffu, al, i) + ck * 16;
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_addr(place(i, ck))), "l"(src), "r"(i < in ? 16 : 0) : "memory");
        }
    } else {
#pragma unroll 1
        for (int i = i1; i < 16; i += per) {
            const char * src = reinterpret_cast<const char *>(__shfl_sync(0xffffffffu, al, i)) + ck * 16;
            char *       to  = place(i, ck);
#pragma unroll 1
            for (int e = 0; e < 16; e += esz) {
                if (esz == 4) {
                    *reinterpret_cast<uint32_t *>(to + e) = i < in ? *reinterpret_cast<const uint32_t *>(src + e) : 0u;
                } else {
                    *reinterpret_cast<uint16_t *>(to + e) = i < in ? *reinterpret_cast<const uint16_t *>(src + e) : (uint16_t) 0;
                }
            }
        }
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
    __syncwarp();
    if constexpr (PARTS == 1) {
        if (p.scale < 0.0f) {  // (the maximum of a row's scores is taken before they are multiplied)
#pragma unroll 1
            for (int i = lane / chunks; i < 16; i += per) {
                uint4 * at = reinterpret_cast<uint4 *>(place(i, ck));
                *at        = make_uint4(at->x ^ 0x80008000u, at->y ^ 0x80008000u, at->z ^ 0x80008000u, at->w ^ 0x80008000u);
            }
        }
        if (lane < 16) {
            factors[ra + lane] = by;
        }
    } else {
        // a row with an infinity or NaN becomes zeros with a factor of NaN
        const float sign = p.scale < 0.0f ? -1.0f : 1.0f;
        const int   e0 = lane * E;
#pragma unroll 1
        for (int i0 = 0; i0 < 16; i0 += 4) {
            float    x[4][E];
            uint32_t top[4];
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const char * at = place(i0 + i, e0 * esz / 16) + e0 * esz % 16;
                top[i] = 0;
#pragma unroll
                for (int e = 0; e < E; e += 2) {
                    float2 f;
                    if (esz == 4) {
                        f = reinterpret_cast<const float2 *>(at)[e / 2];
                    } else {
                        const uint32_t u = reinterpret_cast<const uint32_t *>(at)[e / 2];
                        f = p.q.type == KV_F16 ? h2_to_f2(u) : bf2_to_f2(u);
                    }
                    x[i][e] = f.x, x[i][e + 1] = f.y;
                    top[i]  = max(top[i], max(__float_as_uint(f.x) & 0x7fffffffu, __float_as_uint(f.y) & 0x7fffffffu));
                }
            }
#pragma unroll
            for (int i = 0; i < 4; i++) {
                top[i] = __reduce_max_sync(0xffffffffu, top[i]);  // (and the rows have been read)
            }
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const bool  odd = top[i] >= 0x7f800000u;
                // the row's largest element: F16 to [2^14, 2^15), where its remainders are no small numbers, BF16 to [1, 2) (4)
                const int   ex  = BF16 ? (top[i] == 0 || odd ? 0 : min(max((int) (top[i] >> 23) - 127, -126), 126)) :
                                         (top[i] == 0 || odd ? 0 : max((int) (top[i] >> 23) - 127, -112)) - 14;
                const float dn  = __uint_as_float((uint32_t) (127 - ex) << 23) * sign;
                uint32_t    hi[E / 2], lo[E / 2], third[E / 2];
#pragma unroll
                for (int e = 0; e < E; e += 2) {
                    const float a = odd ? 0.0f : x[i][e] * dn, b = odd ? 0.0f : x[i][e + 1] * dn;
                    hi[e / 2]      = ts_pack<BF16>(a, b);
                    const float2 f = ts_unpack<BF16>(hi[e / 2]);
                    lo[e / 2]      = ts_pack<BF16>(a - f.x, b - f.y);
                    if (PARTS == 3) {
                        const float2 g = ts_unpack<BF16>(lo[e / 2]);
                        third[e / 2]   = ts_pack<BF16>(a - f.x - g.x, b - f.y - g.y);
                    }
                }
                char * to = qs + (e0 / 64) * BLOCK + (ra + i0 + i) * 128 + ((((e0 % 64) / 8) ^ ((i0 + i) & 7)) << 4) + (e0 % 8) * 2;
#pragma unroll
                for (int e = 0; e < E / 2; e++) {
                    reinterpret_cast<uint32_t *>(to)[e]      = hi[e];
                    reinterpret_cast<uint32_t *>(to + QT)[e] = lo[e];
                    if (PARTS == 3) {
                        reinterpret_cast<uint32_t *>(to + 2 * QT)[e] = third[e];
                    }
                }
                if (lane == 0) {
                    factors[ra + i0 + i] = odd ? NAN : __uint_as_float((uint32_t) (127 + ex) << 23) * by;
                }
            }
        }
    }
}

// Waits for the next piece that warp 0 tells of (the first is there since the block's barrier); false: there is none, or it did not come in time.  By whole warps.
__device__ __forceinline__ bool ts_take(const TsPiece * told, uint64_t * bar, uint32_t pieces, uint64_t deadline) {
    const uint32_t k = pieces % TS_PIECES;
    return (pieces == 0 || dn_wait_warp(&bar[TB_PIECE + k], (pieces / TS_PIECES) & 1, deadline)) && told[k].rows > 0;
}

// What warp 0 told is not needed any more.
__device__ __forceinline__ void ts_drop(uint64_t * bar, uint32_t pieces, int lane) {
    __syncwarp();
    if (lane == 0) {
        dn_mbar_arrive(&bar[TB_PFREE + pieces % TS_PIECES]);
    }
}

template <int D, bool BF16, int PARTS>
__global__ void __launch_bounds__(TS_THREADS, 1)
    tree_attn_tc_kernel(const __grid_constant__ CUtensorMap tmk, const __grid_constant__ CUtensorMap tmv, const TreeAttnParams p, int wide,
                        int groups, int slot_rows, int joined) {
    using L          = TsSmem<D, PARTS>;
    constexpr int NS = L::NS, N = L::N;
    extern __shared__ __align__(16) char smem_raw[];
    char *     smem      = smem_raw + ((1024u - (smem_addr(smem_raw) & 1023u)) & 1023u);
    uint64_t * bar       = reinterpret_cast<uint64_t *>(smem + L::OFF_BAR);
    uint32_t * tmem_slot = reinterpret_cast<uint32_t *>(smem + L::OFF_MISC);
    int *      abort_f   = reinterpret_cast<int *>(smem + L::OFF_MISC + 4);
    int *      dirty     = reinterpret_cast<int *>(smem + L::OFF_MISC + 8);  // [4 pieces] a V row of a node held what is no number
    float *    factors   = reinterpret_cast<float *>(smem + L::OFF_F);
    float2 *   ml        = reinterpret_cast<float2 *>(smem + L::OFF_ML);
    uint32_t * anc       = reinterpret_cast<uint32_t *>(smem + L::OFF_ANC);
    int *      par       = reinterpret_cast<int *>(smem + L::OFF_PAR);

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, wg = warp >> 2;
    if (tid == 0) {
        for (int i = 0; i < TB_COUNT; i++) {
            mbar_init(&bar[i], ts_arrivals(i));
        }
        *abort_f = 0, dirty[0] = 0, dirty[1] = 0, dirty[2] = 0, dirty[3] = 0;
        fence_mbar_init();
    }
    if (warp == 1) {
        tmem_alloc(tmem_slot, TS_TMEM);
        tmem_relinquish();
    }
    kv8_dep_wait();
    if (joined) {  // the joining kernel may take its place; it waits for this one's end
        asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    }
    const uint64_t deadline = global_timer_ns() + p.timeout_ns;
    TsPiece *      told = reinterpret_cast<TsPiece *>(smem + L::OFF_PIECE);
    TsPiece        it;
    uint32_t       pieces = 0;  // that a warp has taken
    TsPlan<N>      plan(p, wide, ts_slot_floats(slot_rows, D));
    if (warp == 0) {
        plan.find(groups);
        told[0] = plan.next();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;

    if (wg == 0) {
        regs_dec<TS_REGS_ISSUE>();
        bool ok = true;
        auto next = [&] {
            if (!ok || !ts_take(told, bar, pieces, deadline)) {
                return false;
            }
            it = told[pieces % TS_PIECES];
            ts_drop(bar, pieces, lane);
            return true;
        };
        if (warp == 0) {
            // =================================================== the pieces, TMA
            TsJoin * join = reinterpret_cast<TsJoin *>(reinterpret_cast<char *>(p.status) + TS_SPACE) + blockIdx.x;
            if (lane == 0) {
                uint32_t c = 0;
                join->parts = 0;
                do {
                    if (pieces == 0) {
                        it = told[0];
                    } else {
                        it = plan.next();
                        if (pieces >= (uint32_t) TS_PIECES && !mbar_wait_bounded(&bar[TB_PFREE + pieces % TS_PIECES], (pieces / TS_PIECES - 1) & 1, deadline)) {
                            ok = false;
                            break;
                        }
                        told[pieces % TS_PIECES] = it;
                    }
                    dn_mbar_arrive(&bar[TB_PIECE + pieces % TS_PIECES]);
                    pieces++;
                    if (it.rows == 0) {
                        break;
                    }
                    if (it.a == 0 && it.b < it.tiles) {
                        *join = plan.join(it);
                    }
                    // K(a), K(a + 1), V(a), .., K(b - 1), V(b - 2), V(b - 1)
                    const int n = it.b - it.a;
#pragma unroll 1
                    for (int i = 0; i < 2 * n; i++) {
                        const bool          isk  = i == 0 || ((i & 1) && (i + 1) / 2 < n);
                        const int           tile = it.a + (isk ? (i + 1) / 2 : i == 2 * n - 1 ? n - 1 : i / 2 - 1), slot = (int) (c % NS);
                        const CUtensorMap * tm   = isk ? &tmk : &tmv;
                        if (c >= (uint32_t) NS && !mbar_wait_bounded(&bar[TB_EMPTY + slot], (c / NS - 1) & 1, deadline)) {
                            ok = false;
                            break;
                        }
                        mbar_arrive_expect_tx(&bar[TB_FULL + slot], (uint32_t) L::KT);
#pragma unroll
                        for (int hf = 0; hf < L::HALVES; hf++) {
                            ts_load(smem + L::OFF_RING + slot * L::KT + hf * (N * 128), tm, hf * 64, tile * N, it.h, it.s, &bar[TB_FULL + slot]);
                        }
                        c++;
                    }
                } while (ok);
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
            const uint32_t id_qk = ts_idesc(BF16, N, false), id_pv = ts_idesc(BF16, D, true);
            const uint64_t q_d = sw128_desc(smem_addr(smem + L::OFF_Q), 16, 1024), k_d = sw128_desc(smem_addr(smem + L::OFF_RING), 16, 1024);
            const uint64_t v_d = sw128_desc(smem_addr(smem + L::OFF_RING), (uint32_t) (N * 128), 1024);
            auto wait = [&](int b, uint32_t i) {
                if (ok && !dn_wait_warp(&bar[b], i & 1, deadline)) {
                    ok = false;
                }
                tc_fence_after();
            };
            uint32_t c = 0, tc = 0, looks = 0;
            while (next()) {
                wait(TB_QREADY + (int) (pieces & 1), pieces >> 1);
                pieces++;
#pragma unroll 1
                for (int j = it.a - 1; j < it.b; j++) {  // QK(j + 1), then P V(j)
                    if (j + 1 < it.b) {
                        const int slot = (int) (c % NS), buf = (int) ((tc + (j >= it.a ? 1 : 0)) & 1);
                        wait(TB_FULL + slot, c / NS);
#pragma unroll 1
                        for (int part = PARTS - 1; part >= 0; part--) {
                            uint64_t qa = q_d + (uint64_t) ((part * L::QT) >> 4), kb = k_d + (uint64_t) ((slot * L::KT) >> 4);
#pragma unroll
                            for (int hf = 0; hf < L::HALVES; hf++) {
#pragma unroll
                                for (int k = 0; k < 4; k++) {
                                    umma_f16(tmem + (uint32_t) (buf * TS_S), qa + (uint64_t) (2 * k), kb + (uint64_t) (2 * k), id_qk,
                                             PARTS - 1 - part + hf + k > 0 ? 1u : 0u);
                                }
                                qa += (TS_M * 128) >> 4, kb += (N * 128) >> 4;
                            }
                        }
                        umma_commit(&bar[TB_EMPTY + slot]);
                        umma_commit(&bar[TB_SFULL + buf]);
                        c++;
                        if (j + 2 == it.b) {
                            umma_commit(&bar[TB_QFREE]);
                        }
                    }
                    if (j < it.a) {
                        continue;
                    }
                    const int slot = (int) (c % NS), buf = (int) (tc & 1);
                    wait(TB_FULL + slot, c / NS);
                    const bool nodes = (j + 1) * N > it.L;
                    if (nodes && lane == 0) {
                        dn_mbar_arrive(&bar[TB_LOOK]);
                    }
                    wait(TB_PREADY + buf, tc >> 1);  // (the stream has read the P V of its tile before)
                    if (nodes) {
                        wait(TB_FIX, looks++);
                    }
#pragma unroll 1
                    for (int part = PARTS - 1; part >= 0; part--) {
                        // P of 16 keys: 8 columns, then 8 of its remainder; a second remainder behind them all
                        const uint32_t pa = tmem + (uint32_t) (buf * TS_S + (part == 2 ? N : part * 8)), keys16 = PARTS == 1 || part == 2 ? 8u : 16u;
                        uint64_t vb = v_d + (uint64_t) ((slot * L::KT) >> 4);
                        uint32_t add = PARTS >= 2 ? (uint32_t) (PARTS - 1 - part) : j - it.a < 2 ? 0u : 1u;
#pragma unroll
                        for (int k = 0; k < N / 16; k++) {
                            umma_f16_ts(tmem + 256u + (uint32_t) (buf * D), pa + (uint32_t) k * keys16, vb + (uint64_t) ((k * 16 * 128) >> 4),
                                        id_pv, add);
                            add = 1u;
                        }
                    }
                    umma_commit(&bar[TB_EMPTY + slot]);
                    if (PARTS >= 2 || j + 2 >= it.b) {
                        umma_commit(&bar[TB_OFULL + buf]);
                    }
                    c++, tc++;
                }
            }
            // every product issued has to be complete before TMEM and shared memory are given up
            umma_commit(&bar[TB_DONE]);
            dn_wait_warp(&bar[TB_DONE], 0, global_timer_ns() + p.timeout_ns);
        } else {
            // =================================================== V rows of tiles that hold nodes, and the next piece's Q
            const int t64 = tid - 64;
            uint32_t  c = 0, looks = 0;
            while (next()) {
                const int n = it.b - it.a;
                if (pieces > 0) {
                    if (ok && !dn_wait_warp(&bar[TB_QFREE], (pieces - 1) & 1, deadline)) {
                        ok = false;
                    }
                    // (what lies in rows behind the piece's stays: nothing of theirs is kept.  48 sequences of 52 rows: 355 us, 418)
#pragma unroll 1
                    for (int ra = (warp & 1) * 16; ra < it.rows; ra += 32) {
                        ts_stage16<D, BF16, PARTS, 1>(p, it, ra, smem + L::OFF_Q, factors + (pieces & 1) * TS_M, lane);
                    }
                    fence_proxy_async_smem();
                    dn_mbar_arrive(&bar[TB_QREADY + (pieces & 1)]);
                }
#pragma unroll 1
                for (int j = max(it.a, it.L / N); j < it.b; j++) {
                    const uint32_t i    = c + (uint32_t) (2 * (j - it.a) + (j + 1 < it.b ? 2 : 1));  // its place in the ring's order
                    const int      slot = (int) (i % NS);
                    // (warp 1 has seen the tile land and keeps its place until it is looked at, so that the second wait
                    // finds the phase it names)
                    if (ok && (!dn_wait_warp(&bar[TB_LOOK], looks & 1, deadline) || !dn_wait_warp(&bar[TB_FULL + slot], (i / NS) & 1, deadline))) {
                        ok = false;
                    }
                    char *    tile = smem + L::OFF_RING + slot * L::KT;
                    // A thread has the same 16 bytes of every STEP-th row.  One more in an exponent of ones alone sets the
                    // bit above it, which is how a word's halves are told from numbers (compared one by one: 2 us a tile, and
                    // the product and the next piece's Q wait for this).
                    constexpr int      PER_ROW = 8 * L::HALVES, STEP = 64 / PER_ROW;
                    constexpr uint32_t EXP = BF16 ? 0x7f807f80u : 0x7c007c00u, ONE = BF16 ? 0x00800080u : 0x04000400u;
                    const int          ck = t64 % PER_ROW, end = min(it.keys - j * N, N);
                    char *             col = tile + (ck >> 3) * (N * 128) + (ck & 7) * 16;
                    const int          first = max(0, it.L - j * N) + t64 / PER_ROW;
                    bool               odd = false;
#pragma unroll 1
                    for (int row = first; row < end; row += 4 * STEP) {
                        uint32_t no = 0;
#pragma unroll
                        for (int k = 0; k < 4; k++) {  // (past the end: the row is looked at once more)
                            const uint4 u = *reinterpret_cast<const uint4 *>(col + (row + k * STEP < end ? row + k * STEP : row) * 128);
                            no |= ((u.x & EXP) + ONE) | ((u.y & EXP) + ONE) | ((u.z & EXP) + ONE) | ((u.w & EXP) + ONE);
                        }
                        if (no & 0x80008000u) {
                            odd = true;
#pragma unroll 1
                            for (int k = 0; k < 16 && row + (k >> 2) * STEP < end; k++) {
                                uint32_t * at = reinterpret_cast<uint32_t *>(col + (row + (k >> 2) * STEP) * 128) + (k & 3);
                                *at &= ~__vcmpeq2(*at & EXP, EXP);
                            }
                        }
                    }
#pragma unroll 1
                    for (int row = first + max(0, (end - first + STEP - 1) / STEP) * STEP; row < N; row += STEP) {
                        *reinterpret_cast<uint4 *>(col + row * 128) = make_uint4(0, 0, 0, 0);
                    }
                    if (odd) {
                        atomicExch(&dirty[pieces & 3], 1);
                    }
                    fence_proxy_async_smem();
                    dn_mbar_arrive(&bar[TB_FIX]);
                    looks++;
                }
                c += (uint32_t) (2 * n);
                pieces++;
            }
        }
        if (!ok) {
            atomicExch(abort_f, 1);
        }
    } else {
        // ======================================================= softmax and sums
        regs_inc<TS_REGS_SOFTMAX>();
        const int      w = wg - 1, quad = warp & 3, r = quad * 32 + lane, own = tid - 128;
        const uint32_t tl    = (uint32_t) (quad * 32) << 16;
        const uint32_t s_col = tmem + tl + (uint32_t) (w * TS_S), o_col = tmem + tl + 256u + (uint32_t) (w * D);
        const bool     cap = p.softcap > 0.0f;
        float4 *       turn = reinterpret_cast<float4 *>(smem + L::OFF_XCH) + w * (TS_M * 4);  // 16 columns of a warp's rows, on their way out
        uint32_t       tc = 0, used = 0;
        bool           ok = true;
        auto           wait = [&](int b, uint32_t i) {
            if (ok && !dn_wait_warp(&bar[b], i & 1, deadline)) {
                ok = false;
            }
            tc_fence_after();
        };
        // (all of them go on, or none: they meet at barriers)
        while (softmax_all(ts_take(told, bar, pieces, deadline))) {
            // (read where it is needed: the sums leave few registers)
            const TsPiece & it = told[pieces % TS_PIECES];
            if (own == 0) {
                // of the piece before, which all have left: that place's next piece, the third from here, cannot have been looked
                // at before all came through the loop's head again
                dirty[(pieces + 3) & 3] = 0;
            }
            const int       tile0 = it.a, tile1 = it.b, held = it.L;
            const int       row = it.rb * TS_M + r, my_node = row / p.ratio;
            const uint32_t * bits = anc + min(my_node, TREE_MAX - 1) * (TREE_MAX / 32);
            const bool      live = r < it.rows, warp_live = quad * 32 < it.rows;
            // ---- Q of the first piece, and each node's ancestors, where the piece has tiles with nodes
            const bool tail = tile1 * N > held;
            {
                const int nodes = it.nodes, parent = tail && own < nodes ? tree_parent(p.t, it.s % p.t.n_tree, own) : -1;
                if (pieces == 0) {
                    ts_stage16<D, BF16, PARTS, 4>(p, it, (w * 4 + quad) * 16, smem + L::OFF_Q, factors, lane);
                    fence_proxy_async_smem();
                    __syncwarp();
                    if (lane < 8) {
                        dn_mbar_arrive(&bar[TB_QREADY]);
                    }
                }
                if (tail) {
                    if (own < nodes) {
                        par[own] = parent;
                    }
                    softmax_barrier();
                    if (own < nodes) {
                        uint32_t * to = anc + own * (TREE_MAX / 32);
#pragma unroll
                        for (int k = 0; k < TREE_MAX / 32; k++) {
                            to[k] = 0;
                        }
#pragma unroll 1
                        for (int at = own; at >= 0; at = par[at]) {
                            to[at >> 5] |= held + at < p.n_kv ? 1u << (at & 31) : 0u;
                        }
                    }
                    softmax_barrier();
                }
            }
            wait(TB_QREADY + (int) (pieces & 1), pieces >> 1);
            // What a score is multiplied by is above 0 and finite: 0 by the -inf of a key that is not seen, and an infinity by a
            // score of 0, would be no number.  (Where scale and q's powers of two give a product below 2^-149, the scores are 0 in effect)
            const float f0 = factors[(pieces & 1) * TS_M + r], fx = f0 != f0 ? 1.0f : fminf(fmaxf(f0, 0x1p-149f), TS_MOST), factor = cap ? 1.0f : fx;
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
                    return ((1u << -o) - 1u) | bits[0] << -o;
                }
                const uint32_t lo = bits[o >> 5], hi = o + 32 < TREE_MAX ? bits[(o >> 5) + 1] : 0u;
                return __funnelshift_r(lo, hi, o & 31);
            };
            float m = -INFINITY, l = 0.0f, acc[PARTS >= 2 ? D : 1];
            bool  any = false;  // the stream has a tile of the piece
            if constexpr (PARTS >= 2) {
#pragma unroll
                for (int e = 0; e < D; e++) {
                    acc[e] = 0.0f;
                }
            }
#pragma unroll 1
            for (int j = tile0; j < tile1; j++, tc++) {
                if ((int) (tc & 1) != w) {
                    continue;
                }
                wait(TB_SFULL + w, tc >> 1);
                if (warp_live && cap) {  // over S: s = cap * tanh(S * factor), in log2 units
#pragma unroll 1
                    for (int c = 0; c < N / 16; c++) {
                        uint32_t v[16];
                        tmem_ld16(s_col + (uint32_t) (c * 16), v);
                        tmem_ld16_wait(v);
#pragma unroll
                        for (int e = 0; e < 16; e++) {
                            v[e] = __float_as_uint(ts_tanh(__uint_as_float(v[e]) * fx) * (p.softcap * LOG2E));
                        }
                        tmem_st16(s_col + (uint32_t) (c * 16), v);
                    }
                    tmem_st_wait();
                }
                if (warp_live && (j + 1) * N > held) {  // over S: -inf for a key that the row does not see
#pragma unroll 1
                    for (int c = 0; c < N / 32; c++) {
                        uint32_t v[32];
                        tmem_ld32(s_col + (uint32_t) (c * 32), v);
                        const uint32_t see = live ? seen(j * N + c * 32) : 0u;
                        tmem_ld_wait_tie(v);
#pragma unroll
                        for (int e = 0; e < 32; e++) {
                            v[e] = see >> e & 1u ? v[e] : 0xff800000u;
                        }
                        tmem_st32(s_col + (uint32_t) (c * 32), v);
                    }
                    tmem_st_wait();
                }
                if constexpr (PARTS == 1) {
                    if (warp_live) {
                        uint32_t v[N];
#pragma unroll
                        for (int c = 0; c < 4; c++) {
                            tmem_ld32(s_col + (uint32_t) (c * 32), &v[c * 32]);
                        }
#pragma unroll
                        for (int c = 0; c < 4; c++) {
                            tmem_ld_wait_tie(&v[c * 32]);
                        }
                        float a = __uint_as_float(v[0]), b = __uint_as_float(v[1]);
#pragma unroll
                        for (int e = 2; e < N - 2; e += 4) {
                            a = fmax3(a, __uint_as_float(v[e]), __uint_as_float(v[e + 1]));
                            b = fmax3(b, __uint_as_float(v[e + 2]), __uint_as_float(v[e + 3]));
                        }
                        const float top = fmaxf(fmax3(a, __uint_as_float(v[N - 2]), __uint_as_float(v[N - 1])), b);
                        const float mn   = fmaxf(m, top * factor);
                        const bool  grew = mn > m + (float) TS_GROW;  // (at first too)
                        if (any && __any_sync(0xffffffffu, grew)) {
                            // P V(j - 2) is complete: QK(j) was issued after it
                            const float g = grew ? ex2(m - mn) : 1.0f;
                            l *= g;
#pragma unroll 1
                            for (int c = 0; c < D / 16; c++) {
                                uint32_t o[16];
                                tmem_ld16(o_col + (uint32_t) (c * 16), o);
                                tmem_ld16_wait(o);
#pragma unroll
                                for (int e = 0; e < 16; e++) {
                                    o[e] = __float_as_uint(__uint_as_float(o[e]) * g);
                                }
                                tmem_st16(o_col + (uint32_t) (c * 16), o);
                            }
                        }
                        m = grew ? mn : m;
                        const float    nm = (m == -INFINITY ? 0.0f : -m) + TS_OFF<BF16, PARTS>;
                        const uint64_t nm2 = f2pack(nm, nm), fa2 = f2pack(factor, factor);
                        uint64_t       sum2 = 0ull;
#pragma unroll
                        for (int c = 0; c < 4; c++) {
                            uint32_t hi[16];
#pragma unroll
                            for (int i = 0; i < 16; i++) {
                                float x, y;
                                f2unpack(ffma2(f2pack(__uint_as_float(v[c * 32 + 2 * i]), __uint_as_float(v[c * 32 + 2 * i + 1])), fa2, nm2), x, y);
                                const uint64_t p2 = f2pack(ex2(x), ex2(y));
                                sum2 = fadd2(sum2, p2);
                                f2unpack(p2, x, y);
                                hi[i] = ts_pack<BF16>(x, y);
                            }
                            tmem_st16(s_col + (uint32_t) (c * 16), hi);
                        }
                        float x, y;
                        f2unpack(sum2, x, y);
                        l += x + y;
                        tmem_st_wait();
                    }
                    any = true;
                    tc_fence_before();
                    dn_mbar_arrive(&bar[TB_PREADY + w]);
                } else {
                    float g = 1.0f;
                    if (warp_live) {
                        float top = -INFINITY;
#pragma unroll 1
                        for (int c = 0; c < N / 32; c++) {
                            uint32_t v[32];
                            tmem_ld32(s_col + (uint32_t) (c * 32), v);
                            tmem_ld_wait_tie(v);
                            float a = __uint_as_float(v[0]), b = __uint_as_float(v[1]);
#pragma unroll
                            for (int e = 2; e < 30; e += 4) {
                                a = fmax3(a, __uint_as_float(v[e]), __uint_as_float(v[e + 1]));
                                b = fmax3(b, __uint_as_float(v[e + 2]), __uint_as_float(v[e + 3]));
                            }
                            top = fmax3(top, fmax3(a, __uint_as_float(v[30]), __uint_as_float(v[31])), b);
                        }
                        const float mn = fmaxf(m, top * factor);
                        g = m == mn ? 1.0f : ex2(m - mn);
                        m = mn;
                        const float    nm = (m == -INFINITY ? 0.0f : -m) + TS_OFF<BF16, PARTS>;
                        const uint64_t nm2 = f2pack(nm, nm), fa2 = f2pack(factor, factor);
                        uint64_t       sum2 = 0ull;
                        // 16 columns and the load of the next ones; over them 8 of the weights' first part and 8 of the second
                        uint32_t v[2][16];
                        auto     weights = [&](uint32_t (&s16)[16], int c) {
                            uint32_t hi[16], third[8];
#pragma unroll
                            for (int i = 0; i < 8; i++) {
                                float x, y;
                                f2unpack(ffma2(f2pack(__uint_as_float(s16[2 * i]), __uint_as_float(s16[2 * i + 1])), fa2, nm2), x, y);
                                const uint64_t p2 = f2pack(ex2(x), ex2(y));
                                sum2 = fadd2(sum2, p2);
                                f2unpack(p2, x, y);
                                // the remainder of a weight above 0 is above 0, so that its product with an infinite value has
                                // the sign of the other part's (2^-38 of the row's largest weight is far below F32's last bit)
                                hi[i] = ts_pack_rz<BF16>(x, y);
                                const float2 f = ts_unpack<BF16>(hi[i]);
                                const uint32_t least = __vminu2(hi[i], BF16 ? 0x00800080u : 0x00010001u);
                                f2unpack(ffma2(f2pack(f.x, f.y), f2pack(-1.0f, -1.0f), p2), x, y);
                                if constexpr (PARTS == 3) {
                                    const uint32_t mid = ts_pack_rz<BF16>(x, y);
                                    const float2   g   = ts_unpack<BF16>(mid);
                                    hi[8 + i] = __vmaxu2(mid, least);
                                    third[i]  = __vmaxu2(ts_pack<BF16>(x - g.x, y - g.y), least);
                                } else {
                                    hi[8 + i] = __vmaxu2(ts_pack<BF16>(x, y), least);
                                }
                            }
                            tmem_st16(s_col + (uint32_t) (c * 16), hi);
                            if constexpr (PARTS == 3) {
                                tmem_st8(s_col + (uint32_t) (N + c * 8), third);
                            }
                        };
                        tmem_ld16(s_col, v[0]);
                        tmem_ld16_wait(v[0]);
#pragma unroll 1
                        for (int c = 0; c < N / 16; c += 2) {
                            tmem_ld16(s_col + (uint32_t) (c * 16 + 16), v[1]);
                            weights(v[0], c);
                            tmem_ld16_wait(v[1]);
                            if (c + 2 < N / 16) {
                                tmem_ld16(s_col + (uint32_t) (c * 16 + 32), v[0]);
                            }
                            weights(v[1], c + 1);
                            tmem_ld16_wait(v[0]);
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
                            for (int e = 0; e < 32; e += 2) {
                                f2unpack(ffma2(f2pack(acc[c * 32 + e], acc[c * 32 + e + 1]), f2pack(g, g), f2pack(__uint_as_float(o[e]), __uint_as_float(o[e + 1]))),
                                         acc[c * 32 + e], acc[c * 32 + e + 1]);
                            }
                        }
                    }
                }
            }
            // ---- the two streams' maxima and sums
            if constexpr (PARTS >= 2) {  // to where PARTS 1 has them
#pragma unroll
                for (int c = 0; c < D / 32; c++) {
                    uint32_t o[32];
#pragma unroll
                    for (int e = 0; e < 32; e++) {
                        o[e] = __float_as_uint(acc[c * 32 + e]);
                    }
                    tmem_st32(o_col + (uint32_t) (c * 32), o);
                }
                tmem_st_wait();
            }
            ml[w * TS_M + r] = make_float2(m, l);
            if (PARTS == 1 && any) {
                wait(TB_OFULL + w, used++);
            }
            tc_fence_before();
            softmax_barrier();
            tc_fence_after();
            const float2 other = ml[(w ^ 1) * TS_M + r];
            const float  M = fmaxf(m, other.x), mine_f = m == M ? 1.0f : ex2(m - M), other_f = other.x == M ? 1.0f : ex2(other.x - M);
            l = w == 0 ? fmaf(l, mine_f, other.y * other_f) : fmaf(other.y, other_f, l * mine_f);
            l = f0 != f0 && M != -INFINITY ? NAN : l;
            const float inv = l != 0.0f ? 1.0f / l : 0.0f;
            const bool  whole = tile0 == 0 && tile1 == it.tiles;
            uint64_t    al;  // where this row goes, or the part's slot
            if (whole) {
                const int hd = it.h * p.ratio + row - my_node * p.ratio;
                al = reinterpret_cast<uint64_t>(p.o.data + (int64_t) hd * p.o.nb1 + (int64_t) my_node * p.o.nb2 + (int64_t) it.s * p.o.nb3);
            } else {
                al = reinterpret_cast<uint64_t>(p.part + it.slot);
            }
            if (!whole && live && w == 0) {  // behind the slot's rows
                reinterpret_cast<float2 *>(al + (int64_t) slot_rows * D * 4)[r] = make_float2(M, l);
            }
            // ---- the sums: each stream takes half of the columns of both, 16 at a time, and stores them by whole rows (a
            // warpgroup's warps reach the lanes of the other's; the loop's head holds the next piece's products back)
            const bool odd = tail && dirty[pieces & 3] && live;
            // (PARTS 1: what is there is the piece's where the stream had a tile of it)
            const bool mine_is = PARTS >= 2 || any, theirs_is = PARTS >= 2 || !any || tile1 - tile0 > 1;
            const int  swz = (r >> 1) & 3;
#pragma unroll 1
            for (int c = 0; c < D / 32; c++) {
                const int mine = w * (D / 2) + c * 16;
                uint32_t  o[16], q[16];
                tmem_ld16(tmem + tl + 256u + (uint32_t) (w * D + mine), o);
                tmem_ld16(tmem + tl + 256u + (uint32_t) ((w ^ 1) * D + mine), q);
                tmem_ld16_wait(o);
                tmem_ld16_wait(q);
                float x[16];
#pragma unroll
                for (int e = 0; e < 16; e++) {
                    x[e] = (mine_is ? __uint_as_float(o[e]) * mine_f : 0.0f) + (theirs_is ? __uint_as_float(q[e]) * other_f : 0.0f);
                }
                if (odd) {
                    // elements that are no numbers, of nodes that the row sees: they were left out of the products
#pragma unroll 1
                    for (int n = 0; n < it.nodes; n++) {
                        const int key = held + n;
                        if (key / N < tile0 || key / N >= tile1 || !(bits[n >> 5] >> (n & 31) & 1u)) {
                            continue;
                        }
                        const uint16_t * v = reinterpret_cast<const uint16_t *>(p.v.data + (int64_t) key * p.v.nb1 + (int64_t) it.h * p.v.nb2 + (int64_t) it.s * p.v.nb3) + mine;
#pragma unroll
                        for (int e = 0; e < 16; e++) {
                            const float y = ts_unpack<BF16>(v[e]).x;
                            x[e] += fabsf(y) < INFINITY ? 0.0f : y;
                        }
                    }
                }
                if (!whole && live) {
#pragma unroll
                    for (int k = 0; k < 4; k++) {
                        reinterpret_cast<float4 *>(al)[(mine / 4 + k) * slot_rows + r] = make_float4(x[4 * k], x[4 * k + 1], x[4 * k + 2], x[4 * k + 3]);
                    }
                }
                if (whole && warp_live) {
#pragma unroll
                    for (int k = 0; k < 4; k++) {
                        turn[r * 4 + (k ^ swz)] = make_float4(x[4 * k] * inv, x[4 * k + 1] * inv, x[4 * k + 2] * inv, x[4 * k + 3] * inv);
                    }
                    __syncwarp();
#pragma unroll 1
                    for (int i = lane >> 2; i < 32; i += 8) {
                        const int    k = lane & 3;
                        const float4 f = turn[(quad * 32 + i) * 4 + (k ^ ((i >> 1) & 3))];
                        char *       to = reinterpret_cast<char *>(__shfl_sync(0xffffffffu, al, i));
                        if (quad * 32 + i < it.rows) {
                            ts_store4(to, mine + k * 4, f, p.o.type, p.o.vec);
                        }
                    }
                    __syncwarp();
                }
            }
            tc_fence_before();
            ts_drop(bar, pieces, lane);
            pieces++;
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

// Joins the parts of a unit, in their order, for 32 rows, a row by each lane, and 4 * COLS columns from c4 on: the loads of
// PER parts in flight.
template <int COLS, int PER>
__device__ __forceinline__ void ts_join(const TreeAttnParams & p, const TsJoin & t, int64_t step, int slot_rows, int D, int r, int c4) {
    float  M = -INFINITY, l = 0.0f;
    float4 o[COLS];
#pragma unroll
    for (int c = 0; c < COLS; c++) {
        o[c] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    }
#pragma unroll 1
    for (int k0 = 0; k0 < t.parts; k0 += PER) {
        float2 x[PER];
        float4 v[PER][COLS];
#pragma unroll
        for (int k = 0; k < PER; k++) {
            x[k] = make_float2(-INFINITY, 0.0f);
            if (k0 + k < t.parts) {
                const float * at = p.part + (k0 + k == 0 ? t.part0 : t.part1 + (k0 + k - 1) * step);
                x[k] = reinterpret_cast<const float2 *>(at + slot_rows * D)[r];
#pragma unroll
                for (int c = 0; c < COLS; c++) {
                    v[k][c] = reinterpret_cast<const float4 *>(at)[(c4 + c) * slot_rows + r];
                }
            }
        }
        float top = M;
#pragma unroll
        for (int k = 0; k < PER; k++) {
            top = fmaxf(top, x[k].x);
        }
        const float g = M == top ? 1.0f : ex2(M - top);
        l *= g, M = top;
#pragma unroll
        for (int c = 0; c < COLS; c++) {
            o[c].x *= g, o[c].y *= g, o[c].z *= g, o[c].w *= g;
        }
#pragma unroll
        for (int k = 0; k < PER; k++) {
            if (k0 + k < t.parts) {
                const float f = x[k].x == M ? 1.0f : ex2(x[k].x - M);
                l = fmaf(x[k].y, f, l);
#pragma unroll
                for (int c = 0; c < COLS; c++) {
                    o[c].x = fmaf(v[k][c].x, f, o[c].x), o[c].y = fmaf(v[k][c].y, f, o[c].y);
                    o[c].z = fmaf(v[k][c].z, f, o[c].z), o[c].w = fmaf(v[k][c].w, f, o[c].w);
                }
            }
        }
    }
    const float inv = l != 0.0f ? 1.0f / l : 0.0f;
    const int   row = (int) t.row0 + r, node = row / p.ratio, head = t.h * p.ratio + row - node * p.ratio;
    char *      to  = p.o.data + (int64_t) head * p.o.nb1 + (int64_t) node * p.o.nb2 + (int64_t) t.s * p.o.nb3;
#pragma unroll
    for (int c = 0; c < COLS; c++) {
        ts_store4(to, 4 * (c4 + c), make_float4(o[c].x * inv, o[c].y * inv, o[c].z * inv, o[c].w * inv), p.o.type, p.o.vec);
    }
}

// The joining kernel.  Every CTA finds the units in parts from what the first kernel's CTAs have left, and takes its share of
// all (a CTA for each of those CTAs and each share of a unit: 2368 of them take longer to come and go than to work).  A warp
// takes 32 rows and four columns of a unit where that gives each warp one turn: few units, of many parts.  Otherwise 16
// columns at a time: the units on a line have two or three parts, and a turn is the wait for its loads.
template <int D>
__global__ void __launch_bounds__(32 * TJ_WARPS, 2) tree_attn_join_kernel(const TreeAttnParams p, int ctas, int wide, int slot_rows) {
    __shared__ int list[TJ_UNITS], counts[TJ_WARPS];
    const int      tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    kv8_dep_wait();
    const TsJoin * units   = reinterpret_cast<const TsJoin *>(reinterpret_cast<const char *>(p.status) + TS_SPACE);
    int            n_units = 0;
    for (int i0 = 0; i0 < ctas; i0 += 32 * TJ_WARPS) {
        const bool     has = i0 + tid < ctas && units[i0 + tid].parts > 0;
        const unsigned all = __ballot_sync(0xffffffffu, has);
        if (lane == 0) {
            counts[warp] = __popc(all);
        }
        __syncthreads();
        int at = n_units + __popc(all & ((1u << lane) - 1u));
#pragma unroll
        for (int w = 0; w < TJ_WARPS; w++) {
            at += w < warp ? counts[w] : 0;
            n_units += counts[w];
        }
        if (has) {
            list[at] = i0 + tid;
        }
        __syncthreads();
    }
    const int     warps = (int) gridDim.x * TJ_WARPS, quarters = (slot_rows + 31) / 32;
    const bool    few   = n_units * quarters * (D / 4) <= warps;
    const int     per_unit = quarters * (few ? D / 4 : D / 16);
    const int64_t step     = (int64_t) wide * 2 * ts_slot_floats(slot_rows, D);
    for (int item = (int) blockIdx.x * TJ_WARPS + warp; item < n_units * per_unit; item += warps) {
        const TsJoin t = units[list[item / per_unit]];
        const int    c = item % per_unit / quarters, r = item % quarters * 32 + lane;
        if (r >= t.rows) {
            continue;
        }
        if (few) {
            ts_join<1, 10>(p, t, step, slot_rows, D, r, c);
        } else {
            ts_join<4, 2>(p, t, step, slot_rows, D, r, 4 * c);
        }
    }
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
    constexpr int smem = TsSmem<D, PARTS>::TOTAL, N = TsSmem<D, PARTS>::N;
    cudaError_t   e    = once.smem(kern, smem);
    if (e != cudaSuccess) {
        return e;
    }
    alignas(64) CUtensorMap tmk, tmv;
    for (CUtensorMap * tm : { &tmk, &tmv }) {
        const Kv8Rows & x = tm == &tmk ? p.k : p.v;
        // (the stride of a slab's only row is never stepped, and may be one that a map does not take)
        if (!encode_kv_tensor_map(tm, x.data, BF16, D, p.n_kv, p.n_head_kv, p.n_seq, p.n_kv > 1 ? x.nb1 : 2 * D, x.nb2, x.nb3, N)) {
            return cudaErrorInvalidValue;
        }
    }
    const int wide = tree_attn_wide(p), groups = tree_attn_groups(p, N, sms);
    const int rows = std::min(p.t.max_nodes * p.ratio, TS_M);
    e = kv8_launch(kern, dim3((unsigned) (groups * wide)), TS_THREADS, smem, stream, tmk, tmv, p, wide, groups, rows, p.n_kv <= TS_LEAST * N ? 0 : 1);
    if (e != cudaSuccess || p.n_kv <= TS_LEAST * N) {
        return e;  // (no unit is in parts)
    }
    const int items = groups * wide * ((rows + 31) / 32) * (D / 4);
    return kv8_launch(tree_attn_join_kernel<D>, dim3((unsigned) std::min((items + TJ_WARPS - 1) / TJ_WARPS, 2 * sms)), 32 * TJ_WARPS, 0, stream, p, groups * wide, wide, rows);
}

template <int D, bool BF16>
cudaError_t launch_d(const TreeAttnParams & p, int sms, cudaStream_t stream) {
    // one part where q is the cache's type, the result has no more bits, and the truncated sums stay small; three where two
    // would not give what an F32 result holds
    if (p.q.type == p.k.type && p.o.type == p.q.type && p.n_kv <= TS_LONG) {
        return launch_one<D, BF16, 1>(p, sms, stream);
    }
    if constexpr (BF16) {
        if (p.o.type == KV_F32) {
            return launch_one<D, BF16, 3>(p, sms, stream);
        }
    }
    return launch_one<D, BF16, 2>(p, sms, stream);
}

}  // namespace

// keys of a tile, at least: the result's type decides, which neither the choice of kernel nor the workspace's size goes by
static int least_keys(const TreeAttnParams & p) {
    return ts_keys(p.k.type == KV_BF16 ? 3 : 2);
}

// 16-bit slabs at D = 64 and 128
bool tree_attn_tc_sizes(const TreeAttnParams & p) {
    return (p.k.type == KV_F16 || p.k.type == KV_BF16) && (p.D == 64 || p.D == 128) && tensor_maps_available() &&
           (int64_t) p.n_seq * p.n_head_kv * ((p.t.max_nodes * p.ratio + TS_M - 1) / TS_M) * ((p.n_kv + least_keys(p) - 1) / least_keys(p) + TS_COST) < (1 << 30);
}

// of these, slabs whose strides a tensor map takes
bool tree_attn_tc_takes(const TreeAttnParams & p) {
    for (const Kv8Rows * x : { &p.k, &p.v }) {
        const int64_t most = (int64_t) 1 << 40;
        if (!x->vec || (p.n_kv > 1 && (x->nb1 < 2 * p.D || x->nb1 >= most)) || (p.n_head_kv > 1 && (x->nb2 <= 0 || x->nb2 >= most)) ||
            (p.n_seq > 1 && (x->nb3 <= 0 || x->nb3 >= most))) {
            return false;
        }
    }
    return tree_attn_tc_sizes(p);
}

int tree_attn_wide(const TreeAttnParams & p) {
    return p.t.n_nodes ? 1 : (p.t.max_nodes * p.ratio + TS_M - 1) / TS_M;
}

int tree_attn_groups(const TreeAttnParams & p, int keys, int sms) {
    const int64_t blocks = (p.t.max_nodes * p.ratio + TS_M - 1) / TS_M, wide = tree_attn_wide(p);
    const int64_t tiles = (int64_t) p.n_seq * p.n_head_kv * ((p.n_kv + keys - 1) / keys) * (wide == 1 ? blocks : 1);
    return (int) std::max<int64_t>(1, std::min<int64_t>(sms / wide, tiles));
}

size_t tree_attn_tc_workspace(const TreeAttnParams & p, int sms) {
    const int rows = std::min(p.t.max_nodes * p.ratio, TS_M);
    return KV8_WS_ZEROED + (size_t) tree_attn_groups(p, least_keys(p), sms) * tree_attn_wide(p) * 2 * ts_slot_floats(rows, p.D) * 4;
}

cudaError_t launch_tree_attn_tc(TreeAttnParams p, int sms, cudaStream_t stream) {
    p.part     = reinterpret_cast<float *>(reinterpret_cast<char *>(p.status) + KV8_WS_ZEROED);
    if (p.D == 64) {
        return p.k.type == KV_BF16 ? launch_d<64, true>(p, sms, stream) : launch_d<64, false>(p, sms, stream);
    }
    return p.k.type == KV_BF16 ? launch_d<128, true>(p, sms, stream) : launch_d<128, false>(p, sms, stream);
}

}  // namespace mm3fa
