// paged_chunk.cuh — attention of chunks of new tokens over a paged cache on
// tcgen05 tensor cores.
//
// A persistent CTA takes units: 256 rows of one (sequence, KV head) - row = (new
// token, query head of the group) - as two tiles of 128, and the keys they see in
// tiles of 128.  Warps:
//   0-3, 4-7  softmax of row tile 0 / 1, a thread per row: scores from TMEM, running
//             maximum and sum in registers, weights back to TMEM (over the scores,
//             in halves, so that the product starts on the first); at the end the
//             rows' results.  A unit of up to 128 rows has one row tile: then both
//             halves work on it, on every second key tile, and join their sums
//             (32 drafted or 12 new tokens over 8,192, 64 sequences, 8 KV heads,
//             D = 128: 472 us -> 392; with the second half idle a tile took as long
//             as two)
//   8         TMA: K and V tiles in turn into a ring of stages, page by page
//             (boxes of up to 128 rows of one page and head; a box that no row sees
//             is asked for out of range and arrives as zeros).  A lane looks up a
//             box's page, 32 boxes ahead of those that are asked for; a tile's pages
//             at a time left the read of the table in the chain (8,192 tokens, pages
//             of 16: 505 -> 478 us)
//   9         MMA issue: S_w = Q_w K^T (both in shared memory), then O_w += P_w V
//             with P_w from TMEM
//   10        zeros over V rows that no row of the CTA sees (a page's end)
//   11        the next unit (from the lengths on the device) and its queries
//   12-15     of a cache in 8 bits: codes from a ring of their own to the stages' 16-bit tiles,
//             zeros over V's unseen rows among them (10 rests).  8,192 tokens, int8: 735 us; what
//             the products, which read shared memory at its full rate, leave is the bound
// Heads of 129 to 256 values: units of one row tile, whose sums take half of TMEM, on
// warps 0-3 and a ring of two stages (2,048 tokens, 16 query and 4 KV heads, D = 256:
// 72 us; by the rows kernel 990).
// While one tile's rows are in the exponentials the tensor cores work on the
// other.  S_w of the next key tile is issued after P_w V of this one, so one
// barrier per tile and direction is enough: scores that are ready imply that
// the sum with the previous weights is complete.  (At D = 64 TMEM has room for
// weights beside the scores, so that the next scores need not wait: 468 us
// against 420; the two halves then keep step and want the same units at once.)
//
// The maximum that the weights refer to is only moved when a row's has grown by
// more than 2^8: weights then stay below 256 (fp16: 2^15; exact in the fp32 sums, a
// common factor in the result), and the sums in TMEM are rescaled rarely.
//
// Bound: 4 D FLOP per (row, key) on the tensor cores, 2,048 clocks for the two row
// tiles and a key tile at D = 128, and as many for their exponentials on the
// special-function units, 16 a clock.  Measured, 32 query and 8 KV heads, 8,192
// tokens, causal: D = 128 455-478 us (1,150-1,210 TFLOP/s, about 4,000 clocks a
// tile; 500-530 in a loop of calls, at the clocks that the power limit leaves); without the exponentials it is no faster, with the products and loads
// alone 418: reading K and V into shared memory, 64 KB a tile and CTA, and their
// reading by both row tiles' products bound it (bytes, not boxes: pages of 128 take 459
// where pages of 16 take 456).  D = 64 422 us (650 TFLOP/s): the
// softmax warps' instructions do; exponentials moved to the FMA pipe only add (1 of
// 8: 437).
#pragma once

#include <algorithm>

#include "paged_attn.cuh"
#include "paged_attn_tc.cuh"
#include "paged_code_tile.cuh"

namespace hmm {
namespace serve {
using namespace sm100;

constexpr int TC_ROWS = 128;                 // rows of a tile (MMA M, TMEM lanes)
constexpr int TC_TILES = 2;
static_assert(TC_CTA_ROWS == TC_ROWS * TC_TILES, "a unit is its row tiles");
constexpr int TC_KEYS = 128;                 // keys of a tile
constexpr int TC_SOFTMAX_WARPS = 8;          // two row tiles, 32 rows a warp
constexpr int TC_WIDEN_WARPS = 4;            // a cache in 8 bits: codes to 16-bit tiles
template <int C>
__host__ __device__ constexpr int tc_threads() { return 32 * (TC_SOFTMAX_WARPS + 4 + (C == CODEC_NONE ? 0 : TC_WIDEN_WARPS)); }
// Registers: 384 threads are launched with 168 each (64,512 in all); the softmax warps
// take 224 (a row's scores stay in registers), the last warpgroup keeps 56.  512 threads are
// launched with 128 (65,536): the softmax warps take 208, the others 48.
template <int C>
__host__ __device__ constexpr int tc_regs_launch() { return C == CODEC_NONE ? 168 : 128; }
template <int C>
__host__ __device__ constexpr int tc_regs_softmax() { return C == CODEC_NONE ? 224 : 208; }
template <int C>
__host__ __device__ constexpr int tc_regs_other() { return C == CODEC_NONE ? 56 : 48; }
constexpr int TC_MIN_PIECE = 3;              // key tiles of a piece, at least
constexpr int TC_UNIT_COST = 3;              // key tiles that a unit's start and end take the time of
// Units are cut when they are fewer than the CTAs (at 1.4 a CTA, a mixed step, cut took 121 us
// and whole ones 106) and the longest is longer than an equal share by what the join costs, in
// key tiles: 128 units of 2,000 tokens, a window of 1,024 (D = 64) took 55 us cut and 43 whole,
// 64 units of 512 tokens over 4,096 (D = 128) 64 cut and 81 whole.
constexpr int TC_JOIN_COST = 10;
constexpr float TC_GROWTH = 8.0f;            // log2 of the growth that moves a row's maximum
// log2 of what weights are held by, beside that growth: fp16 ends at 2^16 and 2^-25, so the
// largest are 2^15, and keys far below the largest keep a weight.
template <typename T>
__host__ __device__ constexpr float tc_up() { return std::is_same<T, __half>::value ? 7.0f : 0.0f; }

// Rows of a unit: at D = 256 the sums of one row tile take the TMEM beside its scores, and
// the second half of the softmax warps rests.
template <int DP>
__host__ __device__ constexpr int tc_rows() { return DP == 256 ? TC_ROWS : TC_CTA_ROWS; }
template <int DP, int C>
__host__ __device__ constexpr int tc_stages() {
    return C == CODEC_NONE ? (DP == 64 ? 8 : DP == 128 ? 5 : 2) : DP == 64 ? 6 : DP == 128 ? 4 : 2;
}
// A cache in 8 bits: the ring of codes and scale bytes as they lie in the cache, a tile's keys a
// stage (D = 256: half of them).
template <int DP>
__host__ __device__ constexpr int tc_code_keys() { return DP == 256 ? TC_KEYS / 2 : TC_KEYS; }
template <int DP>
__host__ __device__ constexpr int tc_code_stages() { return DP == 64 ? 6 : 2; }
template <int DP>
__host__ __device__ constexpr int tc_code_bytes() { return tc_code_keys<DP>() * (DP + DP / Q_GROUP); }
template <int DP>
__host__ __device__ constexpr int tc_tile_bytes() { return TC_KEYS * DP * 2; }
template <int DP>
__host__ __device__ constexpr int tc_q_bytes() { return tc_rows<DP>() * DP * 2; }

struct TcArgs {
    AttnArgs a;
    int rows_log2;       // rows of a unit
    int min_rows;        // sequences of fewer rows are another kernel's
    int box_rows;        // rows of a TMA box: a power of two that divides page_tokens
    int split;           // whether few units may be cut into pieces
    int q_tokens;        // new tokens of a row tile's TMA box, 0: queries by 16-byte copies
    uint64_t wait_ns;    // limit of a bounded wait for one step: copies, products, weights of a tile
    uint64_t unit_ns;    // and of one for the end of a unit, or of the two before it
    uint32_t* again;     // [units][TC_SOFTMAX_WARPS] rows of finite scores that came out not finite
    int units;           // sequences that overlap (a cu_new that descends) would be more units
    ChunkJoin join;
};

// What a CTA works on at a time: 256 (D = 256: 128) rows of a (sequence, KV head) and `n` key tiles of
// those that they see, from the t0-th on.
struct Unit {
    int s, kvh, row0, rows;      // s < 0: no more
    Seq q;
    Span sp;
    int sink_tiles, first;       // the seen tiles are [0, sink_tiles) and [first, ...)
    int t0, n, n_of[TC_TILES];   // key tiles of each row tile, a prefix of the unit's; alone: of each half
    bool alone;                  // one row tile: both halves of the softmax warps work on it, on every second key tile
    int slot, id;                // where a piece's sums go (-1: the unit is whole); the unit's number
    __device__ __forceinline__ int key0(int j) const {
        return (t0 + j < sink_tiles ? t0 + j : first + t0 + j - sink_tiles) * TC_KEYS;
    }
    // tiles with keys that no row sees beside some that are seen
    __device__ __forceinline__ bool mends(int k0) const {
        return !(k0 >= sp.lo && k0 + TC_KEYS <= sp.hi) && k0 + TC_KEYS > sp.sink;
    }
};

// The plan of a launch, the same for every CTA: with units for several rounds each CTA
// takes whole ones; fewer are laid end to end and cut into equal pieces, one per CTA.
struct Plan {
    int64_t per, tiles;          // per = 0: whole units
};

template <int DP>
struct TcCtrl {
    uint64_t full[8], empty[8];
    uint64_t c_full[6], c_empty[6];   // (codes)
    uint64_t s_full[TC_TILES], p_full[TC_TILES][2], o_free[TC_TILES];
    uint64_t u_full[2], u_empty[2], q_full, q_empty, v_mend, v_fixed, o_full, drain, half_full;
    float2 half[DP == 256 ? 1 : TC_ROWS];   // alone: the second half's maxima (log2) and sums
    Unit unit[2];
    Plan plan;
    int any_again;
    uint32_t tmem;
    int abort;
};
template <int DP, int C>
__host__ __device__ constexpr size_t tc_smem() {
    return tc_q_bytes<DP>() + tc_stages<DP, C>() * tc_tile_bytes<DP>() +
           (C == CODEC_NONE ? 0 : tc_code_stages<DP>() * tc_code_bytes<DP>()) + sizeof(TcCtrl<DP>);
}

template <int N>
__device__ __forceinline__ void set_regs_up() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N)); }
template <int N>
__device__ __forceinline__ void set_regs_down() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N)); }

// All warps, between the roles and what follows.  No warp may take registers
// back before it: the softmax warps might still be waiting for them.
template <int C>
__device__ __forceinline__ void roles_done() {
    asm volatile("barrier.cta.sync 1, %0;" ::"n"(tc_threads<C>()) : "memory");
}

__device__ __forceinline__ bool wait_warp(uint64_t* bar, uint32_t parity, volatile int* abort, uint64_t ns) {
    return __all_sync(0xffffffffu, mbar_wait_bounded(bar, parity, abort, ns));
}

// One box of the queries: values [x, x + 64) of heads y... of tokens z....
__device__ __forceinline__ void tma_load_q(uint32_t dst, const CUtensorMap* map, uint64_t* bar, int x, int y, int z) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes"
        " [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(dst),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(smem_u32(bar)), "r"(x), "r"(y), "r"(z)
        : "memory");
}

// One CTA's kind::f16 MMAs with the descriptors' halves apart: the upper words are
// constants and the lower ones differ by constants (addresses are below 2^18, so a
// descriptor's address field never carries), which leaves the issuing thread one
// addition per operand.  D[tmem] (+)= A[smem] x B[smem] and D (+)= A[tmem] x B[smem].
// One lane of the warp issues (`one`); the warp's flow stays uniform, so that the
// operands are computed once per warp.
__device__ __forceinline__ void mma_ss(uint32_t one, uint32_t d, uint32_t alo, uint32_t ahi, uint32_t blo,
                                       uint32_t bhi, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p, e;\n\t.reg .b64 da, db;\n\t"
        "mov.b64 da, {%1, %2};\n\tmov.b64 db, {%3, %4};\n\t"
        "setp.ne.b32 p, %6, 0;\n\tsetp.ne.b32 e, %7, 0;\n\t"
        "@e tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %5, p;\n\t}" ::"r"(d),
        "r"(alo), "r"(ahi), "r"(blo), "r"(bhi), "r"(idesc), "r"(accumulate), "r"(one)
        : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t one, uint32_t d, uint32_t a, uint32_t blo, uint32_t bhi,
                                       uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p, e;\n\t.reg .b64 db;\n\t"
        "mov.b64 db, {%2, %3};\n\t"
        "setp.ne.b32 p, %5, 0;\n\tsetp.ne.b32 e, %6, 0;\n\t"
        "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], db, %4, p;\n\t}" ::"r"(d),
        "r"(a), "r"(blo), "r"(bhi), "r"(idesc), "r"(accumulate), "r"(one)
        : "memory");
}
__device__ __forceinline__ void commit_one(uint32_t one, uint64_t* bar) {
    asm volatile(
        "{\n\t.reg .pred e;\n\tsetp.ne.b32 e, %1, 0;\n\t"
        "@e tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(
            smem_u32(bar)),
        "r"(one)
        : "memory");
}
__device__ __forceinline__ void tmem_st_x32(uint32_t taddr, const uint32_t* v) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
        "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,"
        "%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(taddr),
        "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]),
        "r"(v[8]), "r"(v[9]), "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]),
        "r"(v[15]), "r"(v[16]), "r"(v[17]), "r"(v[18]), "r"(v[19]), "r"(v[20]), "r"(v[21]),
        "r"(v[22]), "r"(v[23]), "r"(v[24]), "r"(v[25]), "r"(v[26]), "r"(v[27]), "r"(v[28]),
        "r"(v[29]), "r"(v[30]), "r"(v[31])
        : "memory");
}
__device__ __forceinline__ void tmem_st_x16(uint32_t taddr, const uint32_t* v) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(taddr),
        "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]),
        "r"(v[8]), "r"(v[9]), "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15])
        : "memory");
}
__device__ __forceinline__ void tmem_wait_st() {
    asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
}

// Shared-memory descriptor of an MN-major operand (V: keys are the MMA's K, the
// values of a key are contiguous): 128-byte rows of 64 values with the 128-byte
// swizzle, 8 rows 1,024 bytes apart (stride offset), blocks of 64 values
// `block` bytes apart (leading offset), version 1.
__device__ __forceinline__ uint64_t desc_mn_sw128(uint32_t addr, uint32_t block) {
    return (uint64_t)((addr >> 4) & 0x3FFFu) | ((uint64_t)(block >> 4) << 16) |
           ((uint64_t)(1024 >> 4) << 32) | ((uint64_t)1 << 46) | ((uint64_t)2 << 61);
}

__device__ __forceinline__ uint64_t pack_f2(float lo, float hi) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
    return r;
}
__device__ __forceinline__ void unpack_f2(uint64_t v, float& lo, float& hi) {
    asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v));
}
__device__ __forceinline__ uint64_t fma_f2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
    return d;
}
__device__ __forceinline__ uint64_t add_f2(uint64_t a, uint64_t b) {
    uint64_t d;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}

// The largest of three, NaN if one is.
__device__ __forceinline__ float max3(float a, float b, float c) {
    float d;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}

// Weights exp2(sc (s - m) + tc_up) of 64 of a row's scores v, packed in pairs, to TMEM, and their
// sum (two pairs of partial sums), AT of 32 registers at a time (the warps that widen leave
// fewer; 0: they stay in p, for the caller to store); with TOP also the largest of the 128
// scores from v on.
// m = -inf (no key seen yet) gives exp2(sc s).  The maximum (ALU) and what follows a weight (FMA
// and ALU) stand between the exponentials, which keep the special-function unit for 8
// clocks each: apart, the two would take their times in turn.
template <typename T, bool TOP, int AT>
__device__ __forceinline__ float weights(const uint32_t* v, uint64_t sc2, float m, float sc, uint32_t to,
                                         uint32_t* p, uint64_t* sum) {
    constexpr int LAG = 2;   // pairs between a weight's exponential and its use
    const float neg = m == -INFINITY ? 0.0f : fmaf(-m, sc, tc_up<T>());
    const uint64_t neg2 = pack_f2(neg, neg);
    sum[0] = sum[1] = pack_f2(0.0f, 0.0f);
    float x[32], y[32], mx0 = -INFINITY, mx1 = -INFINITY;
#pragma unroll
    for (int i = 0; i < 32 + LAG; ++i) {
        if (i < 32) {
            const uint64_t e = fma_f2(pack_f2(__uint_as_float(v[2 * i]), __uint_as_float(v[2 * i + 1])), sc2, neg2);
            unpack_f2(e, x[i], y[i]);
            x[i] = ex2(x[i]);
            y[i] = ex2(y[i]);
            if (TOP) {
                mx0 = max3(mx0, __uint_as_float(v[4 * i]), __uint_as_float(v[4 * i + 1]));
                mx1 = max3(mx1, __uint_as_float(v[4 * i + 2]), __uint_as_float(v[4 * i + 3]));
            }
        }
        if (i >= LAG) {
            const int u = i - LAG;
            sum[u & 1] = add_f2(sum[u & 1], pack_f2(x[u], y[u]));
            // weights in the cache's type for the product: off by half a step, 2^-8 of a
            // weight (bf16) or 2^-11, as the output's own rounding; the sum keeps fp32
            p[u % (AT == 0 ? 32 : AT)] = pack2<T>(x[u], y[u]);
            if (AT == 16 && u % 16 == 15) tmem_st_x16(to + u - 15, p);
        }
    }
    if (AT == 32) tmem_st_x32(to, p);
    return TOP ? max3(mx0, mx1, mx1) : 0.0f;
}

// The lowest n bits, none for n < 0, all from 32 on.
__device__ __forceinline__ uint32_t below(int n) {
    return n <= 0 ? 0u : n >= 32 ? 0xffffffffu : (1u << n) - 1u;
}

// Row blocks of a sequence.
__device__ __forceinline__ int row_blocks(const TcArgs& t, const Seq& q) {
    const int64_t rows = (int64_t)q.n_new * t.a.group;
    return rows < t.min_rows ? 0 : (int)((rows + (1 << t.rows_log2) - 1) >> t.rows_log2);
}

// The seen key tiles of rows [row0, row1) of a sequence.
struct Tiles {
    Span sp;
    int sink_tiles, first, n;
};

__device__ __forceinline__ Tiles tiles_of(const AttnArgs& a, const Seq& q, int row0, int row1) {
    Tiles x;
    x.sp = tile_span(a, q, row0, row1);
    x.sink_tiles = (x.sp.sink + TC_KEYS - 1) / TC_KEYS;
    x.first = max(x.sp.lo / TC_KEYS, x.sink_tiles);
    x.n = x.sink_tiles + max(0, (x.sp.hi + TC_KEYS - 1) / TC_KEYS - x.first);
    return x;
}

__device__ __forceinline__ int last_row(const TcArgs& t, const Seq& q, int rb) {
    return (int)min((int64_t)(rb + 1) << t.rows_log2, (int64_t)q.n_new * t.a.group);
}

// The length of row block rb's units in the plan: their key tiles behind the unit's own cost.
__device__ __forceinline__ int block_length(const TcArgs& t, const Seq& q, int rb) {
    return TC_UNIT_COST + tiles_of(t.a, q, rb << t.rows_log2, last_row(t, q, rb)).n;
}

// Lane `src`'s sequence, for the warp; lane 0's is sequence s0.
template <bool SHARED>
__device__ __forceinline__ Seq shared_seq(const Seq& q, int s0, int src) {
    Seq x = seq_of(s0 + src, __shfl_sync(0xffffffffu, q.begin, src), __shfl_sync(0xffffffffu, q.n_new, src),
                   __shfl_sync(0xffffffffu, q.kv, src));
    if (!SHARED) return x;
    x.pos0 = __shfl_sync(0xffffffffu, q.pos0, src);
    x.lo = __shfl_sync(0xffffffffu, q.lo, src);
    x.row = __shfl_sync(0xffffffffu, q.row, src);
    x.out = __shfl_sync(0xffffffffu, q.out, src);
    return x;
}

__device__ __forceinline__ int64_t warp_sum(int64_t v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

__device__ __forceinline__ int64_t warp_scan(int64_t v) {
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int64_t w = __shfl_up_sync(0xffffffffu, v, o);
        if ((int)(threadIdx.x & 31) >= o) v += w;
    }
    return v;
}

// One warp.
template <bool SHARED>
__device__ __forceinline__ Plan make_plan(const TcArgs& t) {
    const AttnArgs& a = t.a;
    const int lane = threadIdx.x & 31;
    if (!t.split) return Plan{0, 0};
    int64_t units = 0;
    each_seq<SHARED>(a.b, a.max_kv, lane, 32, a.status, [&](const Seq& q) { units += (int64_t)row_blocks(t, q) * a.hk; });
    // (A shared prefix is a long unit beside many short ones.)
    if (!(SHARED && a.b.shared) && warp_sum(units) >= (int64_t)gridDim.x) return Plan{0, 0};
    int64_t tiles = 0;   // (a few row blocks per CTA at most)
    int longest = 0;
    auto add = [&](const Seq& q, int rb) {
        const int n = block_length(t, q, rb);
        tiles += n;
        longest = max(longest, n);
    };
    for (int s0 = 0; s0 < a.b.n_seq; s0 += 32) {
        const int s = s0 + lane;
        Seq q{};
        if (s < a.b.n_seq) q = load_seq<SHARED>(a.b, a.max_kv, s, a.status);
        const int rb = row_blocks(t, q);
        if (rb > 0) add(q, 0);
        unsigned busy = __ballot_sync(0xffffffffu, rb > 1);
        while (busy) {
            const int src = __ffs(busy) - 1;
            busy &= busy - 1;
            const Seq x = shared_seq<SHARED>(q, s0, src);
            const int n = __shfl_sync(0xffffffffu, rb, src);
            for (int i = 1 + lane; i < n; i += 32) add(x, i);
        }
    }
    tiles = warp_sum(tiles) * a.hk;
    longest = __reduce_max_sync(0xffffffffu, longest);
    const int64_t per = max((int64_t)TC_MIN_PIECE + TC_UNIT_COST, (tiles + gridDim.x - 1) / gridDim.x);
    return longest <= per + TC_JOIN_COST ? Plan{0, 0} : Plan{per, tiles};
}

// Where a CTA has come to: the next tile of its share (cut units), and the 32 sequences where
// its last unit lay, with the tiles or units and the units before them (the order is the
// same for all, so a CTA's next unit is there or behind).
struct Cursor {
    int64_t pos;
    int s0;
    int64_t run, units;
};

// The k-th unit (whole units) or, from c->pos on, the next piece of this CTA's share, into
// *u (s = -1: there is none); moves *c on.  One warp.
template <bool SHARED>
__device__ __forceinline__ void describe(const TcArgs& t, const Plan& plan, int64_t k, Cursor* c, Unit* u) {
    const AttnArgs& a = t.a;
    const int lane = threadIdx.x & 31;
    const int64_t cta = blockIdx.x, ctas = gridDim.x;
    const bool cut = plan.per > 0;
    // Whole units of a sequence fall in size, so rounds go from the first CTA and from the
    // last one in turn.
    const int64_t at = cut ? c->pos : k * ctas + (k & 1 ? ctas - 1 - cta : cta);
    const int64_t end = cut ? min(plan.tiles, (cta + 1) * plan.per) : INT64_MAX;
    int64_t run = c->run, unit_run = c->units;
    for (int s0 = c->s0; s0 < a.b.n_seq && at < end; s0 += 32) {
        c->s0 = s0;
        c->run = run;
        c->units = unit_run;
        const int s = s0 + lane;
        Seq q{};
        if (s < a.b.n_seq) q = load_seq<SHARED>(a.b, a.max_kv, s, a.status);
        const int rb = row_blocks(t, q);
        unsigned busy = __ballot_sync(0xffffffffu, rb > 0);
        if (!cut) {   // past 32 sequences at once
            const int64_t all = warp_sum((int64_t)rb * a.hk);
            if (run + all <= at) {
                run += all;
                continue;
            }
        } else if (!__any_sync(0xffffffffu, rb > 1)) {   // a block each: past them to the one that is meant
            const int64_t v = rb > 0 ? (int64_t)block_length(t, q, 0) * a.hk : 0, incl = warp_scan(v) + run;
            const unsigned here = __ballot_sync(0xffffffffu, incl - v <= at && at < incl);
            const int stop = here ? __ffs(here) - 1 : 32;
            unit_run += (int64_t)__popc(busy & ((stop < 32 ? 1u << stop : 0u) - 1u)) * a.hk;
            if (!here) {
                run = __shfl_sync(0xffffffffu, incl, 31);
                continue;
            }
            run = __shfl_sync(0xffffffffu, incl - v, stop);
            busy = 1u << stop;
        }
        while (busy) {
            const int src = __ffs(busy) - 1;
            busy &= busy - 1;
            const Seq x = shared_seq<SHARED>(q, s0, src);
            const int n_rb = __shfl_sync(0xffffffffu, rb, src);
            // a sequence's last rows see the most keys: they go first, so that the short
            // blocks fill the end
            int b = -1, kvh = 0, v0 = 0, n_all = 0;
            if (!cut) {
                const int64_t in = at - run;
                if (in < (int64_t)n_rb * a.hk) {
                    b = n_rb - 1 - (int)(in / a.hk);
                    kvh = (int)(in % a.hk);
                }
                run += (int64_t)n_rb * a.hk;
            } else {
                for (int i0 = 0; i0 < n_rb && b < 0; i0 += 32) {
                    const int n = i0 + lane < n_rb ? block_length(t, x, n_rb - 1 - i0 - lane) : 0;
                    const int64_t v = (int64_t)n * a.hk, incl = warp_scan(v) + run;
                    const unsigned here = __ballot_sync(0xffffffffu, incl - v <= at && at < incl);
                    if (here) {
                        const int l = __ffs(here) - 1;
                        const int64_t in = at - __shfl_sync(0xffffffffu, incl - v, l);
                        n_all = __shfl_sync(0xffffffffu, n, l);
                        b = n_rb - 1 - i0 - l;
                        kvh = (int)(in / n_all);
                        v0 = (int)(in - (int64_t)kvh * n_all);
                    }
                    run = __shfl_sync(0xffffffffu, incl, 31);
                }
            }
            if (b < 0) {
                unit_run += (int64_t)n_rb * a.hk;
                continue;
            }
            const int row0 = b << t.rows_log2, row1 = last_row(t, x, b);
            const Tiles all = tiles_of(a, x, row0, row1);
            // A piece is [v0, v1) of the unit's length; its own cost alone is none, and who begins
            // within it begins the unit.
            const int v1 = cut ? v0 + (int)min((int64_t)(n_all - v0), end - at) : 0;
            if (cut) c->pos = at + v1 - v0;
            if (cut && v1 <= TC_UNIT_COST && v1 < n_all) break;
            const bool begins = v0 <= TC_UNIT_COST, whole = !cut || (begins && v1 == n_all);
            const int t0 = cut ? max(0, v0 - TC_UNIT_COST) : 0;
            const int most = cut ? max(0, v1 - TC_UNIT_COST) - t0 : INT_MAX;
            if (lane == 0) {
                u->s = s0 + src;
                u->kvh = kvh;
                u->row0 = row0;
                u->rows = row1 - row0;
                u->q = x;
                u->sp = all.sp;
                u->sink_tiles = all.sink_tiles;
                u->first = all.first;
                u->t0 = t0;
                int n = 0;
#pragma unroll
                for (int w = 0; w < TC_TILES; ++w) {
                    const int r0 = row0 + w * TC_ROWS, r1 = min(row1, r0 + TC_ROWS);
                    int nw = 0;
                    if (r0 < r1) {
                        const int hi = tile_span(a, x, r0, r1).hi;
                        nw = all.sink_tiles + max(0, (hi + TC_KEYS - 1) / TC_KEYS - all.first) - t0;
                        nw = max(0, min(nw, most));
                    }
                    u->n_of[w] = nw;
                    n = max(n, nw);
                }
                u->alone = t.rows_log2 == 8 && row1 - row0 <= TC_ROWS;
                if (u->alone) {
                    u->n_of[0] = (n + 1) / 2;
                    u->n_of[1] = n / 2;
                }
                u->n = n;
                u->slot = whole ? -1 : (int)(2 * cta + begins);
                u->id = (int)(cut ? unit_run + (int64_t)(n_rb - 1 - b) * a.hk + kvh : at);
                if (!whole && begins) {   // its other pieces are the next CTAs' first ones
                    t.join.joint[2 * cta] = make_int4(s0 + src, kvh, b, 1 + (int)((n_all - v1 + plan.per - 1) / plan.per));
                    t.join.joint[2 * cta + 1] = make_int4(x.begin, x.n_new, x.kv, 0);
                }
            }
            __syncwarp();
            return;
        }
        if (cut && c->pos != at) break;   // the share ended in a unit's own cost
    }
    if (lane == 0) u->s = -1;
    __syncwarp();
}

// A full sector (32 bytes) or two halves of one.
__device__ __forceinline__ void store32(void* p, const uint32_t* v, bool whole) {
    if (whole) {
        asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(p), "r"(v[0]), "r"(v[1]), "r"(v[2]),
                     "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7])
                     : "memory");
    } else {
        reinterpret_cast<uint4*>(p)[0] = make_uint4(v[0], v[1], v[2], v[3]);
        reinterpret_cast<uint4*>(p)[1] = make_uint4(v[4], v[5], v[6], v[7]);
    }
}

// Byte of 16-byte piece c of row r of Q: [tile][64 columns][128 rows][128 B], swizzled.
template <int DP>
__device__ __forceinline__ uint32_t q_at(int r, int c) {
    const int rr = r % TC_ROWS;
    return (r / TC_ROWS) * (TC_ROWS * DP * 2) + (c >> 3) * (TC_ROWS * 128) + rr * 128 + (((c & 7) ^ (rr & 7)) * 16);
}

// Codes to (a half of) a tile of T as the tensor cores read it, by one warp of four.  The codes lie in
// boxes of 2^box_log2 rows: the rows' codes, then their scale bytes.  A thread takes 16 codes of a
// row at a time; of a row pair one half of the lanes takes the other row, so that eight
// neighbours' writes (16-byte pieces 0, 2, 4, 6 of a 128-byte row, swizzled by its number)
// meet in no bank.  Rows that `seen` denies become zeros.
// The loop is short on purpose: next to the softmax's straight code, a longer one (all rows
// unrolled) did not stay in the instruction cache, and all roles ran slower (drafted tokens 71 us, 58
// so; a tile takes four warps 900 clocks alone and 3,000 here).
template <typename T, int DP, int C, typename Seen>
__device__ __forceinline__ void widen_rows(const unsigned char* codes, const AttnArgs& a, int box_log2, unsigned char* tile,
                                           int warp, int lane, bool some, Seen seen) {
    constexpr int PIECES = DP / 16, ROWS = 32 / PIECES, STEP = TC_WIDEN_WARPS * ROWS;
    constexpr int AHEAD = 2;                             // rows whose codes are read at once
    static_assert(STEP % 8 == 0 && tc_code_keys<DP>() % (STEP * AHEAD) == 0, "a thread's rows are swizzled alike");
    const int p = lane % PIECES, r0 = (warp * ROWS + lane / PIECES) ^ (PIECES >= 8 ? p >> 2 & 1 : 0);
    const int per = a.quant.per_token, row_bytes = a.D, box_bytes = (row_bytes + per) << box_log2, in_box = (1 << box_log2) - 1;
    const bool real = 16 * p < row_bytes;
    unsigned char* to = tile + (p >> 2) * (TC_KEYS * 128) + r0 * 128;
    const int at0 = ((2 * p & 7) ^ (r0 & 7)) * 16, at1 = at0 ^ 16;
    const unsigned char *row = codes + 16 * p, *scale = codes + (row_bytes << box_log2) + (p >> 1);
#pragma unroll 1
    for (int r = r0; r < tc_code_keys<DP>(); r += AHEAD * STEP, to += AHEAD * STEP * 128) {
        uint4 w[AHEAD];
        uint32_t s[AHEAD];
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) {
            const int x = r + i * STEP, box = (x >> box_log2) * box_bytes, in = x & in_box;
            w[i] = make_uint4(0u, 0u, 0u, 0u);
            s[i] = 127;
            if (real && (!some || seen(x))) {
                w[i] = *reinterpret_cast<const uint4*>(row + box + in * row_bytes);
                s[i] = scale[box + in * per];
            }
        }
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) {
            const uint32_t m = multiplier<T, C>(s[i] * 0x00010001u), u[4] = {w[i].x, w[i].y, w[i].z, w[i].w};
            uint32_t v[8];
#pragma unroll
            for (int x = 0; x < 4; ++x) {
                uint32_t even, odd;
                widen<T, C>(u[x], even, odd);
                even = mul_pair<T>(even, m);
                odd = mul_pair<T>(odd, m);
                v[2 * x] = in_order_lo(even, odd);
                v[2 * x + 1] = in_order_hi(even, odd);
            }
            *reinterpret_cast<uint4*>(to + i * STEP * 128 + at0) = make_uint4(v[0], v[1], v[2], v[3]);
            *reinterpret_cast<uint4*>(to + i * STEP * 128 + at1) = make_uint4(v[4], v[5], v[6], v[7]);
        }
    }
}

// SHARED: the batch may be one of parts (Batch::shared), whose keys begin at Seq::lo and whose rows may go
// to AttnArgs::part.  What that adds to the softmax warps' code is felt where their issue is the bound, so
// a plain batch over 16 bits has a kernel without it (86 bytes of spills for 130; 8,192 tokens, heads of
// 64: 424.5 -> 422 us, heads of 128 as before).
template <typename T, int DP, int C, bool SHARED>
__global__ void __launch_bounds__(tc_threads<C>(), 1)
paged_chunk_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV,
                   const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ TcArgs t) {
    constexpr bool QUANT = C != CODEC_NONE;
    constexpr int ST = tc_stages<DP, C>();
    // codes: stages, a stage's keys and bytes, stages of a tile
    constexpr int CST = tc_code_stages<DP>(), CKEYS = tc_code_keys<DP>(), CODES = tc_code_bytes<DP>(), PARTS = TC_KEYS / CKEYS;
    constexpr int TILE = tc_tile_bytes<DP>();
    constexpr int HALVES = DP / 64;                    // 128-byte column blocks
    constexpr int UNIT = tc_rows<DP>();
    extern __shared__ __align__(1024) unsigned char smem_raw[];
    // The swizzle needs 1,024-byte alignment, which the array's alignment gives (there is
    // no room to round up to it); should it ever not, the call says so.
    if ((smem_u32(smem_raw) & 1023u) != 0) {
        if (threadIdx.x == 0) {
            atomicOr(t.a.status, HMM_STATUS_TIMEOUT);
            if (t.split) t.join.joint[2 * blockIdx.x] = make_int4(0, 0, 0, 0);
        }
        asm volatile("griddepcontrol.wait;" ::: "memory");
        return;
    }
    unsigned char* Qs = smem_raw;                      // [tile][half][128 rows][128 B], swizzled
    unsigned char* Rs = Qs + tc_q_bytes<DP>();         // ring: [stage][half][128 keys][128 B]
    unsigned char* Cs = Rs + ST * TILE;                // codes: [stage][box][rows' codes, their scale bytes]
    TcCtrl<DP>* ctl = reinterpret_cast<TcCtrl<DP>*>(Cs + (QUANT ? CST * CODES : 0));
    const AttnArgs& a = t.a;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    volatile int* abort = &ctl->abort;
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

    if (threadIdx.x == 0) {
        for (int i = 0; i < ST; ++i) {
            mbar_init(&ctl->full[i], QUANT ? TC_WIDEN_WARPS : 1);
            mbar_init(&ctl->empty[i], 1);
        }
        if (QUANT) {
            for (int i = 0; i < CST; ++i) {
                mbar_init(&ctl->c_full[i], 1);
                mbar_init(&ctl->c_empty[i], TC_WIDEN_WARPS);
            }
        }
        for (int w = 0; w < TC_TILES; ++w) {
            mbar_init(&ctl->s_full[w], 1);
            mbar_init(&ctl->p_full[w][0], TC_SOFTMAX_WARPS / 2);
            mbar_init(&ctl->p_full[w][1], TC_SOFTMAX_WARPS / 2);
            mbar_init(&ctl->o_free[w], TC_SOFTMAX_WARPS / 2);
        }
        for (int k = 0; k < 2; ++k) {
            mbar_init(&ctl->u_full[k], 1);
            // softmax, TMA, MMA, zeros or widening
            mbar_init(&ctl->u_empty[k], TC_SOFTMAX_WARPS + 2 + (QUANT ? TC_WIDEN_WARPS : 1));
        }
        mbar_init(&ctl->q_full, 1);
        mbar_init(&ctl->q_empty, 1);
        mbar_init(&ctl->v_mend, 1);
        mbar_init(&ctl->v_fixed, 1);
        mbar_init(&ctl->o_full, 1);
        mbar_init(&ctl->drain, 1);
        mbar_init(&ctl->half_full, TC_SOFTMAX_WARPS / 2);
        ctl->any_again = 0;
        ctl->abort = 0;
        fence_barrier_init();
    }
    if (warp == TC_SOFTMAX_WARPS + 1) {
        tmem_alloc(&ctl->tmem, 512);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = ctl->tmem;   // S_w at 128 w, O_w at 256 + DP w
    auto give_up = [&] {
        if (lane == 0) {
            atomicExch(&ctl->abort, 1);
            atomicOr(a.status, HMM_STATUS_TIMEOUT);
        }
    };
    // The k-th unit lies in ctl->unit[k & 1] between these two.
    auto take = [&](int k) { return wait_warp(&ctl->u_full[k & 1], (k >> 1) & 1, abort, t.unit_ns); };
    auto leave = [&](int k) {
        __syncwarp();
        if (lane == 0) mbar_arrive(&ctl->u_empty[k & 1]);
    };

    // The same setmaxnreg for all warps of a warpgroup; what is outside of the roles runs
    // with the launch's registers again.
    if (warp >= TC_SOFTMAX_WARPS) {
        set_regs_down<tc_regs_other<C>()>();
        if (warp == TC_SOFTMAX_WARPS) {
            // -------------------------------------------------------- producer
            // A lane looks up one box's page: of 32 boxes, that is of `ahead` key tiles, at once,
            // and of the next 32 while these are asked for.
            const int br = t.box_rows, subs = TC_KEYS / br, ahead = 32 / subs;
            if (!QUANT && lane == 0) {
                prefetch_tmap(&tmK);
                prefetch_tmap(&tmV);
            }
            uint32_t i = 0;                                   // boxes' tiles so far, K and V in turn
            bool ok = true;
            for (int k = 0; ok; ++k) {
                const Unit& u = ctl->unit[k & 1];
                if (!(ok = take(k)) || u.s < 0) break;
                const int mine = lane / subs, sub = lane % subs;
                auto lookup = [&](int j, int* page, int* row) {   // lane: box `sub` of tile j + mine
                    *page = a.n_pages;                            // out of range: zeros (-1: of a seen box)
                    *row = 0;
                    if (j + mine < u.n) {
                        const int k0 = u.key0(j + mine) + sub * br;
                        if (k0 < u.sp.sink || (k0 + br > u.sp.lo && k0 < u.sp.hi)) {
                            const int lp = a.by_page(k0), e = page_of(a, u.q.row, lp);
                            if (e >= 0) {
                                *page = e;
                                *row = k0 - lp * a.page_tokens;
                            } else if (QUANT) {
                                *page = -1;
                            }
                        }
                    }
                };
                int page, row;
                lookup(0, &page, &row);
                for (int j0 = 0; ok && j0 < u.n; j0 += ahead) {
                    int next_page, next_row;
                    lookup(j0 + ahead, &next_page, &next_row);
                    const int n = min(ahead, u.n - j0);
                    for (int j = 0; ok && j < n; ++j) {
                        if constexpr (QUANT) {
                            // A box that no row sees is not asked for (K's scores there are masked, V's rows
                            // become zeros); one that is seen, but whose page is out of range, is zeros.
                            const int per = a.quant.per_token, box_bytes = br * (a.D + per);
                            const int64_t in_page = (int64_t)row * a.D, scale_at = a.quant.scales + (int64_t)row * per;
#pragma unroll 1
                            for (int x = 0; x < 2 * PARTS; ++x, ++i) {
                                const uint32_t st = i % CST;
                                const bool here = mine == j && (PARTS == 1 || sub * br / CKEYS == x % PARTS);
                                const bool in = here && (uint32_t)page < (uint32_t)a.n_pages;
                                const Pages& p = x < PARTS ? a.k : a.v;
                                const unsigned char* src = p.base + page * p.page + u.kvh * p.head;
                                unsigned char* to = Cs + st * CODES + (PARTS == 1 ? sub : sub & (CKEYS / br - 1)) * box_bytes;
                                const uint32_t bytes = box_bytes * __popc(__ballot_sync(0xffffffffu, in));
                                if (!(ok = wait_warp(&ctl->c_empty[st], ((i / CST) & 1) ^ 1, abort, t.wait_ns))) break;
                                if (here && page < 0) {
                                    for (int z = 0; z < box_bytes; z += 16)
                                        *reinterpret_cast<uint4*>(to + z) = make_uint4(0u, 0u, 0u, 0u);
                                    fence_proxy_async_smem();   // before the stage's next copies
                                }
                                __syncwarp();
                                if (lane == 0) mbar_expect_tx(&ctl->c_full[st], bytes);
                                __syncwarp();
                                if (!in) continue;
                                const uint32_t dst = smem_u32(to);
                                if (br == a.page_tokens) {   // all of a page and head: one block
                                    bulk_load(dst, src, box_bytes, &ctl->c_full[st]);
                                } else {
                                    bulk_load(dst, src + in_page, br * a.D, &ctl->c_full[st]);
                                    bulk_load(dst + br * a.D, src + scale_at, br * per, &ctl->c_full[st]);
                                }
                            }
                        } else {
                            for (int kv = 0; kv < 2; ++kv, ++i) {
                                const uint32_t st = i % ST;
                                if (!(ok = wait_warp(&ctl->empty[st], ((i / ST) & 1) ^ 1, abort, t.wait_ns))) break;
                                if (lane == 0) mbar_expect_tx(&ctl->full[st], TILE);
                                __syncwarp();
                                if (mine == j) {
                                    const uint32_t dst = smem_u32(Rs + st * TILE) + sub * br * 128;
#pragma unroll
                                    for (int h = 0; h < HALVES; ++h)
                                        tma_load_page(dst + h * (TC_KEYS * 128), kv ? &tmV : &tmK, &ctl->full[st], 64 * h,
                                                      row, u.kvh, page);
                                }
                            }
                        }
                    }
                    page = next_page;
                    row = next_row;
                }
                leave(k);
            }
            if (!ok) give_up();
            constexpr uint32_t RING = QUANT ? CST : ST;
            for (uint32_t b = i > RING ? i - RING : 0; b < i; ++b)   // copies in flight, if another role gave up
                mbar_wait_drain(QUANT ? &ctl->c_full[b % RING] : &ctl->full[b % RING], (b / RING) & 1);
        } else if (warp == TC_SOFTMAX_WARPS + 1) {
            // --------------------------------------------------------- MMA
            constexpr int FMT = std::is_same<T, __nv_bfloat16>::value ? 1 : 0;
            const uint32_t id_qk = idesc_f16(TC_ROWS, TC_KEYS, FMT);
            const uint32_t id_pv = idesc_f16(TC_ROWS, DP, FMT) | (1u << 16);   // B is MN-major
            const uint32_t one = elect_one();
            const uint64_t dk = desc_k_sw128(smem_u32(Rs)), dv = desc_mn_sw128(smem_u32(Rs), TC_KEYS * 128);
            const uint64_t dq = desc_k_sw128(smem_u32(Qs));
            const uint32_t khi = (uint32_t)(dk >> 32), vhi = (uint32_t)(dv >> 32);
            const uint32_t klo = (uint32_t)dk, vlo = (uint32_t)dv, qlo = (uint32_t)dq;
            const uint32_t tm = __shfl_sync(0xffffffffu, tmem, 0);
            auto wait = [&](uint64_t* bar, uint32_t parity) {
                return wait_warp(bar, parity, abort, t.wait_ns);
            };
            auto qk = [&](int w, uint32_t k, int rows) {   // scores w of row tile `rows`
                const uint32_t ql = qlo + rows * (TC_ROWS * DP * 2 / 16), d = tm + 128 * w;
#pragma unroll
                for (int ks = 0; ks < DP / 16; ++ks) {
                    const uint32_t off = ((ks >> 2) * (TC_ROWS * 128) + (ks & 3) * 32) / 16;
                    mma_ss(one, d, ql + off, khi, k + off, khi, id_qk, ks != 0);
                }
                commit_one(one, &ctl->s_full[w]);
            };
            int st = 0, ph = 0;                  // the ring's next tile
            auto next = [&](int& x, int& p) {
                if (++x == ST) {
                    x = 0;
                    p ^= 1;
                }
            };
            int fixed = 0, busy = 0;             // tiles mended; units with keys so far
            int tiles[TC_TILES] = {0, 0};        // key tiles of each row tile so far
            bool ok = true;
            for (int k = 0; ok; ++k) {
                if (!(ok = take(k))) break;
                const Unit& u = ctl->unit[k & 1];
                const int us = __shfl_sync(0xffffffffu, u.s, 0), n = __shfl_sync(0xffffffffu, u.n, 0);
                const bool alone = u.alone;
                const int n_of[2] = {__shfl_sync(0xffffffffu, u.n_of[0], 0), __shfl_sync(0xffffffffu, u.n_of[1], 0)};
                // key tiles with rows that no row sees: found from the first and the last few
                const int t0 = u.t0, sink_tiles = u.sink_tiles, first = u.first;
                const int lo = u.sp.lo, hi = u.sp.hi, sink = u.sp.sink;
                leave(k);
                if (us < 0) break;
                if (n == 0) continue;
                // V_j has arrived and is mended, the results of the unit before have left TMEM
                auto ready = [&](int j) {
                    if (!wait(&ctl->full[st], ph)) return false;
                    const int key0 = (t0 + j < sink_tiles ? t0 + j : first + t0 + j - sink_tiles) * TC_KEYS;
                    if (!QUANT && !(key0 >= lo && key0 + TC_KEYS <= hi) && key0 + TC_KEYS > sink) {
                        if (lane == 0) mbar_arrive(&ctl->v_mend);
                        if (!wait(&ctl->v_fixed, fixed++ & 1)) return false;
                    }
                    return j > 0 || busy == 0 ||
                           (wait(&ctl->o_free[0], (busy - 1) & 1) && wait(&ctl->o_free[1], (busy - 1) & 1));
                };
                // O_w += P_w V, its i-th product, as the halves of P_w arrive
                auto pv = [&](int w, int i, uint32_t v) {
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        if (!wait(&ctl->p_full[w][h], ((w ? tiles[1] : tiles[0]) + i) & 1)) return false;
                        tc_fence_after();
#pragma unroll
                        for (int ks = 4 * h; ks < 4 * h + 4; ++ks)
                            mma_ts(one, tm + 256 + DP * w, tm + 128 * w + 8 * ks, v + ks * 128, vhi, id_pv, i > 0 || ks > 0);
                    }
                    return true;
                };
                if (!(ok = wait(&ctl->q_full, busy & 1) && wait(&ctl->full[st], ph))) break;
                tc_fence_after();
                if (alone) {   // key tile j in scores and sums j & 1, which two tiles on are free again
                    int sk = st, pk = ph;        // the next K
                    for (int j = -2; j < n; ++j) {
                        const int w = j & 1;
                        if (j >= 0) {
                            if (!(ok = ready(j) && pv(w, j >> 1, vlo + st * (TILE / 16)))) break;
                            commit_one(one, &ctl->empty[st]);
                            next(st, ph);
                            next(st, ph);
                        }
                        if (j + 2 >= n) continue;
                        if (!(ok = wait(&ctl->full[sk], pk))) break;
                        tc_fence_after();
                        qk(w, klo + sk * (TILE / 16), 0);
                        commit_one(one, &ctl->empty[sk]);
                        if (j + 3 == n) commit_one(one, &ctl->q_empty);
                        next(sk, pk);
                        if (j == -2) {
                            st = sk;             // V_0
                            ph = pk;
                        }
                        next(sk, pk);
                    }
                    if (!ok) break;
                    commit_one(one, &ctl->o_full);
                    // st is one past K_n: back to it
                    st = sk;
                    ph = pk;
                    tiles[0] += n_of[0];
                    tiles[1] += n_of[1];
                    ++busy;
                    continue;
                }
                {
                    const uint32_t kl = klo + st * (TILE / 16);
#pragma unroll
                    for (int w = 0; w < TC_TILES; ++w)
                        if (n_of[w] > 0) qk(w, kl, w);
                }
                commit_one(one, &ctl->empty[st]);
                if (n == 1) commit_one(one, &ctl->q_empty);
                next(st, ph);
                for (int j = 0; ok && j < n; ++j) {
                    int sk = st, pk = ph;        // K_j+1, behind V_j
                    next(sk, pk);
                    const uint32_t v = vlo + st * (TILE / 16), kl = klo + sk * (TILE / 16);
                    if (!(ok = ready(j))) break;
                    bool k_ready = false;
#pragma unroll
                    for (int w = 0; w < TC_TILES; ++w) {
                        if (j >= n_of[w]) continue;
                        if (!(ok = pv(w, j, v))) break;
                        if (j + 1 < n_of[w]) {
                            if (!k_ready && !(ok = wait(&ctl->full[sk], pk))) break;
                            k_ready = true;
                            qk(w, kl, w);
                        }
                    }
                    if (!ok) break;
                    commit_one(one, &ctl->empty[st]);
                    if (j + 1 < n) {
                        commit_one(one, &ctl->empty[sk]);
                        if (j + 2 == n) commit_one(one, &ctl->q_empty);   // the unit's last scores
                        next(st, ph);
                    } else {
                        commit_one(one, &ctl->o_full);
                    }
                    next(st, ph);
                }
                tiles[0] += n_of[0];
                tiles[1] += n_of[1];
                ++busy;
            }
            if (!ok) give_up();
            commit_one(one, &ctl->drain);        // the MMAs issued end before TMEM is freed
            mbar_wait_drain(&ctl->drain, 0);
            __syncwarp();
        } else if (QUANT && warp >= TC_SOFTMAX_WARPS + 4) {
            // ------------------------------------------- codes to 16-bit tiles
            // V rows that no row of the CTA sees become zeros: a weight of zero times what a slot of nobody
            // holds is only zero then.
            const int mine = warp - TC_SOFTMAX_WARPS - 4, box_log2 = 31 - __clz(t.box_rows);
            uint32_t i = 0, c = 0;               // tiles, and stages of codes so far
            bool ok = true;
            for (int k = 0; ok; ++k) {
                const Unit& u = ctl->unit[k & 1];
                if (!(ok = take(k)) || u.s < 0) break;
                const int n = u.n;
#pragma unroll 1
                for (int j = 0; ok && j < 2 * n; ++j, ++i) {
                    const uint32_t st = i % ST;
                    if (!(ok = wait_warp(&ctl->empty[st], ((i / ST) & 1) ^ 1, abort, t.wait_ns))) break;
                    const int key0 = u.key0(j >> 1);
                    const bool some = (j & 1) && u.mends(key0);
#pragma unroll 1
                    for (int x = 0; x < PARTS; ++x, ++c) {
                        const uint32_t cs = c % CST;
                        if (!(ok = wait_warp(&ctl->c_full[cs], (c / CST) & 1, abort, t.wait_ns))) break;
                        unsigned char* to = Rs + st * TILE + x * CKEYS * 128;
                        widen_rows<T, DP, C>(Cs + cs * CODES, a, box_log2, to, mine, lane, some,
                                             [&](int r) { return span_has(u.sp, key0 + x * CKEYS + r); });
                        __syncwarp();
                        if (lane == 0) mbar_arrive(&ctl->c_empty[cs]);
                    }
                    if (!ok) break;
                    fence_proxy_async_smem();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&ctl->full[st]);
                }
                leave(k);
            }
            if (!ok) give_up();
        } else if (QUANT && warp == TC_SOFTMAX_WARPS + 2) {
            // (the warps that widen see to V's unseen rows)
        } else if (warp == TC_SOFTMAX_WARPS + 2) {
            // ------------------------------------------------ V's unseen rows
            // V rows that no row of the CTA sees, in boxes that were read, become zeros:
            // a weight of zero times what a slot of nobody holds is only zero then.
            // The MMA warp says when such a tile has arrived, and waits: this warp, which
            // skips the others, could not tell a stage's phases apart.
            int mended = 0;
            uint32_t base = 0;                   // the ring's tiles before this unit
            bool ok = true;
            for (int k = 0; ok; ++k) {
                const Unit& u = ctl->unit[k & 1];
                if (!(ok = take(k)) || u.s < 0) break;
                for (int j = 0; j < u.n; ++j) {
                    const int key0 = u.key0(j);
                    const uint32_t st = (base + 2 * j + 1) % ST;
                    if (!u.mends(key0)) continue;
                    if (!(ok = wait_warp(&ctl->v_mend, mended++ & 1, abort, t.unit_ns))) break;
                    for (int r = lane; r < TC_KEYS; r += 32) {
                        const int key = key0 + r, k0 = key - r % t.box_rows;
                        if (!span_has(u.sp, key) &&
                            (k0 < u.sp.sink || (k0 + t.box_rows > u.sp.lo && k0 < u.sp.hi))) {
#pragma unroll
                            for (int c = 0; c < HALVES * 8; ++c)
                                *reinterpret_cast<uint4*>(Rs + st * TILE + (c >> 3) * (TC_KEYS * 128) + r * 128 +
                                                          (c & 7) * 16) = make_uint4(0u, 0u, 0u, 0u);
                        }
                    }
                    fence_proxy_async_smem();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&ctl->v_fixed);
                }
                base += 2 * u.n;
                leave(k);
            }
            if (!ok) give_up();
        } else {
            // -------------------------------------- the units, and their queries
            if (t.split && lane == 0) t.join.joint[2 * blockIdx.x] = make_int4(0, 0, 0, 0);
            const Plan plan = make_plan<SHARED>(t);
            if (lane == 0) ctl->plan = plan;
            Cursor at{(int64_t)blockIdx.x * plan.per, 0, 0, 0};
            int loads = 0;                       // units' queries so far
            bool ok = true;
            for (int k = 0; ok; ++k) {
                if (!(ok = wait_warp(&ctl->u_empty[k & 1], ((k >> 1) & 1) ^ 1, abort, t.unit_ns))) break;
                Unit* u = &ctl->unit[k & 1];
                describe<SHARED>(t, plan, k, &at, u);
                const int s = u->s, n = u->n, row0 = u->row0, rows = u->rows, kvh = u->kvh, begin = u->q.begin;
                __syncwarp();
                if (lane == 0) mbar_arrive(&ctl->u_full[k & 1]);
                if (s < 0) break;
                if (n == 0) continue;
                if (!(ok = wait_warp(&ctl->q_empty, (loads & 1) ^ 1, abort, t.unit_ns))) break;
                ++loads;
                constexpr int CH = DP / 8;
                const uint32_t q0 = smem_u32(Qs);
                if (t.q_tokens > 0) {   // a tile's 128 rows are whole tokens' groups: boxes of them
                    if (lane == 0) mbar_expect_tx(&ctl->q_full, tc_q_bytes<DP>());
                    __syncwarp();
                    const int b = lane;
                    if (b < UNIT / TC_ROWS * HALVES)
                        tma_load_q(q0 + b * (TC_ROWS * 128), &tmQ, &ctl->q_full, 64 * (b % HALVES), kvh * a.group,
                                   begin + a.by_group(row0) + (b / HALVES) * t.q_tokens);
                    continue;
                }
                // (rows behind the unit's keep what was there: they are nobody's)
#pragma unroll 4
                for (int i = lane; i < rows * CH; i += 32) {
                    const int r = i / CH, c = i % CH, x = row0 + r, tok = a.by_group(x), head = x - tok * a.group;
                    cp16(q0 + q_at<DP>(r, c),
                         a.q + (int64_t)(begin + tok) * a.q_token + (int64_t)(kvh * a.group + head) * a.q_head +
                             (c * 8 < a.D ? 16 * c : 0),
                         c * 8 < a.D);
                }
                cp_commit();
                cp_wait<0>();
                if (a.scale < 0.0f) {   // turned signs: the largest score is the largest product
#pragma unroll 1
                    for (int i = lane; i < rows * CH; i += 32) {
                        uint4* x = reinterpret_cast<uint4*>(Qs + q_at<DP>(i / CH, i % CH));
                        *x = make_uint4(x->x ^ 0x80008000u, x->y ^ 0x80008000u, x->z ^ 0x80008000u, x->w ^ 0x80008000u);
                    }
                }
                fence_proxy_async_smem();
                __syncwarp();
                if (lane == 0) mbar_arrive(&ctl->q_full);
            }
            if (!ok) give_up();
            if (loads > 0) mbar_wait_drain(&ctl->q_full, (loads - 1) & 1);   // (as the producer's)
        }
        tc_fence_before();
        roles_done<C>();
        set_regs_up<tc_regs_launch<C>()>();   // the softmax warps have given theirs back
    } else {
        // --------------------------------------------------------- softmax
        set_regs_up<tc_regs_softmax<C>()>();
        const int w = warp >> 2;
        const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
        const uint32_t ts = tmem + 128 * w + lanes, to = tmem + 256 + DP * w + lanes;
        const float sc = fabsf(a.scale_log2);
        const uint64_t sc2 = pack_f2(sc, sc);
        int tiles = 0, busy = 0;                               // key tiles, units with keys so far
        bool ok = true;
        for (int k = 0; ok; ++k) {
            const Unit& u = ctl->unit[k & 1];
            if (!(ok = take(k)) || u.s < 0) break;
            // (what the loop does not need is read from the unit again behind it: registers)
            auto row = [&] { return 32 * (u.alone ? warp & 3 : warp) + lane; };   // the thread's of the unit
            const int pos = row_pos(a, u.q, u.row0 + min(row(), u.rows - 1));
            float m = -INFINITY;
            uint64_t l2[2] = {pack_f2(0.0f, 0.0f), pack_f2(0.0f, 0.0f)};
            bool fine = true;
            for (int j = 0; j < u.n_of[w]; ++j) {
                if (!(ok = wait_warp(&ctl->s_full[w], (tiles + j) & 1, abort, t.wait_ns))) break;
                tc_fence_after();
                uint32_t v[TC_KEYS];
#pragma unroll
                for (int c = 0; c < TC_KEYS; c += 32) tmem_ld_x32(ts + c, v + c);
                tmem_wait_ld();
                const int key0 = u.key0(u.alone ? 2 * j + w : j), kv = u.q.kv;
                const int pos_first = __shfl_sync(0xffffffffu, pos, 0), pos_last = __shfl_sync(0xffffffffu, pos, 31);
                if (!(key0 + TC_KEYS <= kv && (!a.causal || key0 + TC_KEYS - 1 <= pos_first) &&
                      (a.window > 0 ? key0 > pos_last - a.window || key0 + TC_KEYS <= a.sinks : !SHARED || key0 >= u.q.lo))) {
                    const int hi = (a.causal ? min(kv, pos + 1) : kv) - key0;
                    const int lo = (a.window > 0 ? max(0, pos - a.window + 1) : SHARED ? u.q.lo : 0) - key0;
                    const int sink = a.window > 0 ? a.sinks - key0 : 0;
#pragma unroll
                    for (int c0 = 0; c0 < TC_KEYS; c0 += 32) {
                        const uint32_t seen = below(hi - c0) & (~below(lo - c0) | below(sink - c0));
#pragma unroll
                        for (int c = 0; c < 32; ++c)
                            if (!((seen >> c) & 1u)) v[c0 + c] = 0xff800000u;
                    }
                }
                // The first half's weights with the maximum so far, while this tile's is found:
                // that is right unless the row grew by more than TC_GROWTH, which is rare.
                // NaN and +inf show in the maximum: such a row is NaN.
                // (They go over the scores, which are in registers, and are written again if it was not.)
                // Stored before the vote below the weights are in TMEM sooner (32/8 heads of 128, 2,048 tokens:
                // 59.2 -> 57.9 us); at D = 64, where these warps' issue is the bound, behind it (8,192 tokens:
                // 429 -> 422 us).
                constexpr int AT = QUANT ? 16 : DP == 64 ? 0 : 32;
                uint64_t sum[2];
                uint32_t p[AT == 0 ? 32 : AT];
#pragma unroll 1
                while (true) {
                    const float top = weights<T, true, AT>(v, sc2, m, sc, ts, p, sum);
                    fine = fine && top < INFINITY;
                    const bool grow = (top - m) * sc > TC_GROWTH && top < INFINITY;
                    if (!__any_sync(0xffffffffu, grow)) break;
                    const float al = grow ? ex2((m - top) * sc) : 1.0f;
                    if (grow) m = top;
                    const uint64_t al2 = pack_f2(al, al);
                    l2[0] = fma_f2(l2[0], al2, pack_f2(0.0f, 0.0f));
                    l2[1] = fma_f2(l2[1], al2, pack_f2(0.0f, 0.0f));
                    if (j > 0) {
#pragma unroll 1
                        for (int c = 0; c < DP; c += 32) {
                            uint32_t o[32];
                            tmem_ld_x32(to + c, o);
                            tmem_wait_ld();
#pragma unroll
                            for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * al);
                            tmem_st_x32(to + c, o);
                        }
                        tmem_wait_st();
                    }
                }
                // the first half's product starts while the second half is in the exponentials
                l2[0] = add_f2(l2[0], sum[0]);
                l2[1] = add_f2(l2[1], sum[1]);
                if (AT == 0) tmem_st_x32(ts, p);
                tmem_wait_st();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&ctl->p_full[w][0]);
                weights<T, false, AT>(v + 64, sc2, m, sc, ts + 32, p, sum);
                if (AT == 0) tmem_st_x32(ts + 32, p);
                l2[0] = add_f2(l2[0], sum[0]);
                l2[1] = add_f2(l2[1], sum[1]);
                tmem_wait_st();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&ctl->p_full[w][1]);
            }
            // ---- the rows' results
            const int n = u.n, nw = u.n_of[w], rows = u.rows, r = row();
            const bool alone = u.alone;
            if (ok && n > 0) ok = wait_warp(&ctl->o_full, busy & 1, abort, t.unit_ns);
            if (!ok) break;
            tc_fence_after();
            tiles += nw;
            float l, lb;
            unpack_f2(add_f2(l2[0], l2[1]), l, lb);
            l += lb;
            const bool live = r < rows && !(alone && w == 1), whole_unit = u.slot < 0;
            bool some = m != -INFINITY, other = false;   // whether this half saw a key, and the other one did
            float top = some ? fmaf(m, sc, -tc_up<T>()) : -INFINITY, s0 = 1.0f, s1 = 0.0f;
            fine = fine && (!some || l > 0.0f);          // (no sum of a maximum's weights: NaN, or scores beyond fp32)
            if (n > 0 && w == 1) {
                if (alone) ctl->half[r] = make_float2(top, fine ? l : NAN);
                __syncwarp();
                if (lane == 0) mbar_arrive(&ctl->half_full);
            } else if (n > 0) {
                if (!(ok = wait_warp(&ctl->half_full, busy & 1, abort, t.unit_ns))) break;
                if (alone) {   // the halves' sums over different keys
                    const float2 x = ctl->half[r];
                    const float both = fmaxf(top, x.x);
                    fine = fine && x.y == x.y;
                    other = x.x != -INFINITY;
                    s0 = some ? ex2(top - both) : 0.0f;
                    s1 = other ? ex2(x.x - both) : 0.0f;
                    l = fmaf(l, s0, x.y * s1);
                    top = both;
                }
            }
            if (!fine) {                                 // every column and lse
                some = true;
                s0 = l = NAN;
            }
            const int x = u.row0 + (live ? r : 0), tok = a.by_group(x), head = x - tok * a.group;
            const int64_t orow = (int64_t)((SHARED ? u.q.out : u.q.begin) + tok) * a.hq + u.kvh * a.group + head;
            float* pt = t.join.part + (int64_t)u.slot * UNIT * (DP + 2);   // (pieces)
            if (whole_unit && l != 0.0f) {
                const float inv = 1.0f / l;
                s0 *= inv;
                s1 *= inv;
            }
            const bool sectors = ((a.D & 15) | (reinterpret_cast<uintptr_t>(a.out) & 31)) == 0;
            uint32_t most = 0;   // an infinity or NaN has the largest bits behind the sign
#pragma unroll 1
            for (int c0 = 0; c0 < (alone && w == 1 ? 0 : DP); c0 += 32) {
                uint32_t o[32];
                if (nw > 0) {
                    tmem_ld_x32(to + c0, o);
                    tmem_wait_ld();
                }
#pragma unroll
                for (int c = 0; c < 32; ++c) o[c] = some ? __float_as_uint(__uint_as_float(o[c]) * s0) : 0u;
                if (alone && u.n_of[1] > 0) {
#pragma unroll
                    for (int h = 0; h < 32; h += 8) {
                        uint32_t o1[8];
                        tmem_ld_x8(to + DP + c0 + h, o1);
                        tmem_wait_ld();
#pragma unroll
                        for (int c = 0; c < 8; ++c)
                            if (other)
                                o[h + c] = __float_as_uint(fmaf(__uint_as_float(o1[c]), s1, __uint_as_float(o[h + c])));
                    }
                }
#pragma unroll
                for (int c = 0; c < 32; ++c) most = max(most, o[c] & 0x7fffffffu);
                if (!live) continue;
                if (!whole_unit) {   // [DP / 4][row][4]: neighbouring rows' quads are neighbours
#pragma unroll
                    for (int c = 0; c < 32; c += 4)
                        *reinterpret_cast<uint4*>(pt + ((c0 + c) / 4 * UNIT + r) * 4) =
                            make_uint4(o[c], o[c + 1], o[c + 2], o[c + 3]);
                    continue;
                }
                if (SHARED && a.part) {
#pragma unroll
                    for (int c = 0; c < 32; c += 8)
                        if (c0 + c < a.D) store32(a.part + orow * a.D + c0 + c, o + c, false);
                    continue;
                }
#pragma unroll
                for (int c = 0; c < 32; c += 16) {
                    uint32_t h[8];
#pragma unroll
                    for (int e = 0; e < 8; ++e)
                        h[e] = pack2<T>(__uint_as_float(o[c + 2 * e]), __uint_as_float(o[c + 2 * e + 1]));
                    unsigned char* dst = a.out + 2 * (orow * a.D + c0 + c);
                    if (c0 + c + 16 <= a.D) store32(dst, h, sectors);
                    else if (c0 + c < a.D) *reinterpret_cast<uint4*>(dst) = make_uint4(h[0], h[1], h[2], h[3]);
                }
            }
            if (n > 0) {
                tc_fence_before();
                __syncwarp();
                if (lane == 0 && !(alone && w == 1)) mbar_arrive(&ctl->o_free[w]);
                if (lane == 0 && alone && w == 0) mbar_arrive(&ctl->o_free[1]);   // (both read by this half)
                ++busy;
            }
            if (live) {
                if (!whole_unit) {
                    // an infinite maximum joins to NaN
                    pt[UNIT * DP + r] = fine ? top : INFINITY;
                    pt[UNIT * (DP + 1) + r] = l;
                } else if (a.lse) {
                    a.lse[orow] = l == 0.0f ? -INFINITY : (top + log2f(l)) * LN2;
                }
            }
            const unsigned again = __ballot_sync(0xffffffffu, live && fine && !(SHARED && a.part) && most >= 0x7f800000u);
            if (lane == 0 && whole_unit && (uint32_t)u.id < (uint32_t)t.units) {
                t.again[(int64_t)u.id * TC_SOFTMAX_WARPS + warp] = again;
                if (again) ctl->any_again = 1;
            }
            leave(k);
        }
        if (!ok) give_up();
        set_regs_down<tc_regs_launch<C>()>();
        tc_fence_before();
        roles_done<C>();
    }
    tc_fence_after();
    if (warp == TC_SOFTMAX_WARPS + 1) tmem_dealloc(tmem, 512);
    if (warp == 0) asm volatile("griddepcontrol.wait;" ::: "memory");   // the rows kernel may still run: not done before it
    // Rows of finite scores that came out not finite, from the definition.
    if (*abort || !ctl->any_again || warp >= TC_SOFTMAX_WARPS) return;
    Unit* u = reinterpret_cast<Unit*>(smem_raw) + warp;   // (nothing is left in the rings)
    const Plan plan = ctl->plan;
    Cursor at{(int64_t)blockIdx.x * plan.per, 0, 0, 0};
    for (int64_t k = 0;; ++k) {
        describe<SHARED>(t, plan, k, &at, u);
        const int s = u->s, kvh = u->kvh, row0 = u->row0 + 32 * warp, slot = u->slot;
        const int id = u->id;
        const Seq q = u->q;
        __syncwarp();
        if (s < 0) break;
        if (slot >= 0 || (uint32_t)id >= (uint32_t)t.units) continue;
        // rows [32 warp, 32 warp + 32) of the unit
        attn_rows_exact<T, C, QUANT ? 4 : 16>(a, q, kvh, row0, __ldcg(t.again + (int64_t)id * TC_SOFTMAX_WARPS + warp));
    }
}

inline int unit_rows(int64_t D) { return D <= 128 ? tc_rows<128>() : tc_rows<256>(); }

template <typename T, int DP, int C, bool SHARED>
hmm_status_t launch_chunk(const TcArgs& t, const CUtensorMap& k, const CUtensorMap& v, const CUtensorMap& q,
                          bool behind, cudaStream_t st) {
    static std::atomic<uint64_t> done{0};
    const hmm_status_t s = allow_smem(paged_chunk_kernel<T, DP, C, SHARED>, tc_smem<DP, C>(), &done);
    if (s != HMM_OK) return s;
    return launch(paged_chunk_kernel<T, DP, C, SHARED>, dim3((unsigned)device_sm_count()), tc_threads<C>(), tc_smem<DP, C>(), behind, st,
                  "paged_chunk_kernel", k, v, q, t);
}

template <typename T, int DP, int C>
hmm_status_t choose_chunk(const TcArgs& t, const CUtensorMap& k, const CUtensorMap& v, const CUtensorMap& q, bool behind,
                          cudaStream_t st) {
    if constexpr (C == CODEC_NONE) {
        if (!t.a.b.shared) return launch_chunk<T, DP, C, false>(t, k, v, q, behind, st);
    }
    return launch_chunk<T, DP, C, true>(t, k, v, q, behind, st);
}

template <int C>
hmm_status_t run_chunk(const AttnArgs& a, bool bf16, int min_rows, bool behind, unsigned char* ws, cudaStream_t st,
                       ChunkJoin* join) {
    const int64_t rows = unit_rows(a.D), tokens = (a.b.shared ? 2 : 1) * (int64_t)a.b.n_tokens,
                  units = most_units(a.b.n_seq, tokens, a.group, a.hk, rows);
    HMM_REQUIRE(units < (int64_t(1) << 30), "n_tokens * n_heads is too large for one call");
    unsigned char* joint = ws + up256(4 * (size_t)units * TC_SOFTMAX_WARPS);
    // A tile of 128 rows is a box of the queries where it is whole tokens; a negative scale
    // turns the signs on the way, which a box cannot.
    const bool boxes = a.group <= TC_ROWS && (a.group & (a.group - 1)) == 0 && a.scale >= 0.0f &&
                       (a.hq == 1 || a.q_head > 0) && (a.b.n_tokens == 1 || a.q_token > 0) &&
                       a.q_head < (int64_t(1) << 40) && a.q_token < (int64_t(1) << 40);
    TcArgs t{};
    t.a = a;
    t.rows_log2 = rows == 256 ? 8 : 7;
    t.min_rows = min_rows;
    t.box_rows = box_rows_of(a.page_tokens, C != CODEC_NONE && a.D > 128 ? tc_code_keys<256>() : TC_KEYS);
    t.split = a.b.shared || may_split(a.b.n_tokens, a.group, a.hk, rows);
    t.q_tokens = boxes ? TC_ROWS / a.group : 0;
    t.wait_ns = wait_limit_ns();
    // 16 us a key tile, which takes 2 to 4 (a limit of 0 stays one)
    t.unit_ns = t.wait_ns == 0 ? 0 : t.wait_ns + 2 * ((uint64_t)a.max_kv / TC_KEYS + 4) * 16000;
    t.again = (uint32_t*)ws;
    t.units = (int)units;
    if (t.split) {
        const int64_t most = std::min<int64_t>(rows, (int64_t)a.b.n_tokens * a.group);
        t.join = ChunkJoin{(int4*)joint, (float*)(joint + up256(2 * sizeof(int4) * device_sm_count())),
                           device_sm_count(), (int)((most + 15) / 16), (int)rows};
    }
    *join = t.join;
    CUtensorMap k{}, v{}, q{};
    hmm_status_t s = HMM_OK;
    if (C == CODEC_NONE) {   // (blocks of codes are copied without a map)
        s = make_page_map(&k, a, a.k, t.box_rows, false);
        if (s == HMM_OK) s = make_page_map(&v, a, a.v, t.box_rows, false);
        if (s != HMM_OK) return s;
    }
    if (boxes) {
        s = make_query_map(&q, a, a.group, TC_ROWS / a.group);
        if (s != HMM_OK) return s;
    }
    if (a.D <= 64)
        return bf16 ? choose_chunk<__nv_bfloat16, 64, C>(t, k, v, q, behind, st)
                    : choose_chunk<__half, 64, C>(t, k, v, q, behind, st);
    if (a.D <= 128)
        return bf16 ? choose_chunk<__nv_bfloat16, 128, C>(t, k, v, q, behind, st)
                    : choose_chunk<__half, 128, C>(t, k, v, q, behind, st);
    return bf16 ? choose_chunk<__nv_bfloat16, 256, C>(t, k, v, q, behind, st)
                : choose_chunk<__half, 256, C>(t, k, v, q, behind, st);
}

}  // namespace serve
}  // namespace hmm
