// paged_attn_tc.cu — attention of chunks of new tokens over a paged cache on
// tcgen05 tensor cores.
//
// A CTA takes 256 rows of one (sequence, KV head) - row = (new token, query head
// of the group) - as two tiles of 128, and the keys they see in tiles of 128:
//   warps 0-7, 8-15 softmax of row tile 0 / 1, two threads per row: scores from
//                   TMEM, running maximum and sum in registers, weights back to
//                   TMEM; at the end the rows' results
//   warp 16         TMA: K and V tiles in turn into a ring of stages, page by
//                   page (boxes of up to 128 rows of one page and head; a box
//                   that no row sees is asked for out of range and arrives as zeros)
//   warp 18         zeros over V rows that no row of the CTA sees (a page's end)
//   warp 17         MMA issue: S_w = Q_w K^T (both in shared memory), then O_w +=
//                   P_w V with P_w from TMEM over S_w's columns
// While one tile's rows are in the exponentials the tensor cores work on the
// other.  S_w of the next key tile is issued after P_w V of this one, so one
// barrier per tile and direction is enough: scores that are ready imply that
// the sum with the previous weights is complete.
//
// The maximum that the weights refer to is only moved when a row's has grown by
// more than 2^8: weights then stay below 256 (exact in the fp32 sums, a common
// factor in the result), and the sums in TMEM are rescaled rarely.
//
// Bound: 4 D FLOP per (row, key) on the tensor cores, against one exponential
// per (row, key) on the special-function units, 16 a clock and SM: at D = 128
// both take 1,024 clocks a tile.
#include <cudaTypedefs.h>

#include <algorithm>
#include <mutex>

#include "paged_attn.cuh"
#include "paged_attn_tc.cuh"

namespace hmm {
namespace serve {
using namespace sm100;
namespace {

constexpr int TC_ROWS = 128;                 // rows of a tile (MMA M, TMEM lanes)
constexpr int TC_TILES = 2;
constexpr int TC_CTA_ROWS = TC_ROWS * TC_TILES;
constexpr int TC_KEYS = 128;                 // keys of a tile
constexpr int TC_SOFTMAX_WARPS = 16;         // two row tiles x 32 rows x two parts of the columns
constexpr int TC_WARPS = TC_SOFTMAX_WARPS + 4;
constexpr int TC_THREADS = 32 * TC_WARPS;
constexpr int TC_SOFTMAX = 32 * TC_SOFTMAX_WARPS;
// Registers: 640 threads are launched with 96 each (61,440 in all); the softmax warps
// take 104 (half a row's scores stay in registers), the last warpgroup gives up to 56.
constexpr int TC_REGS_LAUNCH = 96, TC_REGS_SOFTMAX = 104, TC_REGS_OTHER = 56;
constexpr float TC_GROWTH = 8.0f;            // log2 of the growth that moves a row's maximum

// Of 8 pairs of exponentials, those that go to the FMA pipe.
#ifndef TC_POLY
#define TC_POLY 0
#endif
constexpr float EXP2_C1 = 0.6931470036506653f, EXP2_C2 = 0.24022242426872253f, EXP2_C3 = 0.05550733581185341f,
                EXP2_C4 = 0.009671512991189957f, EXP2_C5 = 0.001326472731307149f;

template <int DP>
__host__ __device__ constexpr int tc_stages() { return DP == 64 ? 8 : 5; }
template <int DP>
__host__ __device__ constexpr int tc_tile_bytes() { return TC_KEYS * DP * 2; }
template <int DP>
__host__ __device__ constexpr int tc_q_bytes() { return TC_CTA_ROWS * DP * 2; }

struct TcCtrl {
    uint64_t full[8], empty[8];
    uint64_t s_full[TC_TILES], p_full[TC_TILES][2], q_full, v_mend, v_fixed, o_full, drain;
    int64_t scan[TC_WARPS];
    int64_t pre;
    Seq own;
    int seq;
    uint32_t tmem;
    uint32_t again[TC_SOFTMAX_WARPS];   // each softmax warp's rows that came out not finite
    float top[2][TC_CTA_ROWS];          // [part][row] a tile's largest scores; at the end sums
    int abort;
};
template <int DP>
__host__ __device__ constexpr size_t tc_smem() {
    return tc_q_bytes<DP>() + tc_stages<DP>() * tc_tile_bytes<DP>() + sizeof(TcCtrl);
}

template <int N>
__device__ __forceinline__ void set_regs_up() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N)); }
template <int N>
__device__ __forceinline__ void set_regs_down() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N)); }

// All warps, between the roles and what follows.  No warp may take registers
// back before it: the softmax warps might still be waiting for them.
__device__ __forceinline__ void roles_done() {
    asm volatile("barrier.cta.sync 1, %0;" ::"n"(TC_THREADS) : "memory");
}

__device__ __forceinline__ bool wait_warp(uint64_t* bar, uint32_t parity, volatile int* abort, uint64_t ns) {
    return __all_sync(0xffffffffu, mbar_wait_bounded(bar, parity, abort, ns));
}

__device__ __forceinline__ void cp16(uint32_t dst, const void* src, bool real) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(real ? 16 : 0)
                 : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

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
__device__ __forceinline__ uint32_t elect_one() {
    uint32_t one;
    asm volatile(
        "{\n\t.reg .pred e;\n\telect.sync _|e, 0xffffffff;\n\tselp.u32 %0, 1, 0, e;\n\t}" : "=r"(one));
    return one;
}

__device__ __forceinline__ void tmem_st_x16(uint32_t taddr, const uint32_t* v) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
        "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(taddr),
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

// 2^x of a pair on the FMA pipe, x <= 2^22: x = n + f with n the nearest whole number
// (read off the low bits of x + 1.5 2^23), 2^f on [-1/2, 1/2] by the polynomial of
// degree 5 with p(0) = 1 that is nearest in relative error (a weighted least-squares
// fit: 2^-23.4), and n added to the exponent.  From -127 down it is 0 (p(0) = 1 makes
// that exact).  A NaN is lost: the caller looks for it in the maximum.
__device__ __forceinline__ void exp2_pair(uint64_t e, float& x, float& y) {
    unpack_f2(e, x, y);
    e = pack_f2(fmaxf(x, -127.0f), fmaxf(y, -127.0f));
    const uint64_t big = pack_f2(12582912.0f, 12582912.0f), nbig = pack_f2(-12582912.0f, -12582912.0f);
    const uint64_t t = add_f2(e, big);
    const uint64_t f = fma_f2(add_f2(t, nbig), pack_f2(-1.0f, -1.0f), e);
    uint64_t p = fma_f2(f, pack_f2(EXP2_C5, EXP2_C5), pack_f2(EXP2_C4, EXP2_C4));
    p = fma_f2(f, p, pack_f2(EXP2_C3, EXP2_C3));
    p = fma_f2(f, p, pack_f2(EXP2_C2, EXP2_C2));
    p = fma_f2(f, p, pack_f2(EXP2_C1, EXP2_C1));
    p = fma_f2(f, p, pack_f2(1.0f, 1.0f));
    float tx, ty;
    unpack_f2(t, tx, ty);
    unpack_f2(p, x, y);
    x = __uint_as_float(__float_as_uint(x) + (__float_as_uint(tx) << 23));
    y = __uint_as_float(__float_as_uint(y) + (__float_as_uint(ty) << 23));
}

// Weights exp2(sc (s - m)) of 32 of a row's scores v, packed in pairs, and their sum (a
// pair of partial sums); with TOP also the largest of the 64 scores from v on.  m = -inf
// (no key seen yet) gives exp2(sc s).  The maximum (ALU) and what follows a weight (FMA
// and ALU) stand between the exponentials, which keep the special-function unit for 8
// clocks each: apart, the two would take their times in turn.
template <typename T, bool TOP>
__device__ __forceinline__ float weights(const uint32_t* v, uint64_t sc2, float m, float sc, uint32_t* p,
                                         uint64_t* sum) {
    constexpr int LAG = 2;   // pairs between a weight's exponential and its use
    const float neg = m == -INFINITY ? 0.0f : -m * sc;
    const uint64_t neg2 = pack_f2(neg, neg);
    uint64_t s0 = pack_f2(0.0f, 0.0f), s1 = s0;
    float x[16], y[16], mx0 = -INFINITY, mx1 = -INFINITY;
#pragma unroll
    for (int i = 0; i < 16 + LAG; ++i) {
        if (i < 16) {
            const uint64_t e = fma_f2(pack_f2(__uint_as_float(v[2 * i]), __uint_as_float(v[2 * i + 1])), sc2, neg2);
            if (i % 8 < TC_POLY) {
                exp2_pair(e, x[i], y[i]);
            } else {
                unpack_f2(e, x[i], y[i]);
                x[i] = ex2(x[i]);
                if (TOP) mx0 = max3(mx0, __uint_as_float(v[4 * i]), __uint_as_float(v[4 * i + 1]));
                y[i] = ex2(y[i]);
            }
            if (TOP && i % 8 < TC_POLY) mx0 = max3(mx0, __uint_as_float(v[4 * i]), __uint_as_float(v[4 * i + 1]));
            if (TOP) mx1 = max3(mx1, __uint_as_float(v[4 * i + 2]), __uint_as_float(v[4 * i + 3]));
        }
        if (i >= LAG) {
            const int u = i - LAG;
            if (u & 1) s1 = add_f2(s1, pack_f2(x[u], y[u]));
            else s0 = add_f2(s0, pack_f2(x[u], y[u]));
            // weights in the cache's type for the product: relative 2^-9 (bf16) or
            // 2^-12, the size of the output's own rounding; the sum keeps fp32
            p[u] = pack2<T>(x[u], y[u]);
        }
    }
    *sum = add_f2(s0, s1);
    return TOP ? max3(mx0, mx1, mx1) : 0.0f;
}

__device__ __forceinline__ void pair_sync(int id) {
    asm volatile("barrier.cta.sync %0, 64;" ::"r"(id) : "memory");
}

// CTAs of a sequence: row blocks x heads.
struct TcLoad {
    int64_t blocks;
    int row_blocks;
};

__device__ __forceinline__ TcLoad tc_load(const TcArgs& t, const Seq& q) {
    const int64_t rows = (int64_t)q.n_new * t.a.group;
    TcLoad x{0, 0};
    if (rows < t.min_rows) return x;
    x.row_blocks = (int)((rows + TC_CTA_ROWS - 1) / TC_CTA_ROWS);
    x.blocks = (int64_t)x.row_blocks * t.a.hk;
    return x;
}

// Byte of 16-byte piece c of row r of Q: [tile][64 columns][128 rows][128 B], swizzled.
template <int DP>
__device__ __forceinline__ uint32_t q_at(int r, int c) {
    const int rr = r % TC_ROWS;
    return (r / TC_ROWS) * (TC_ROWS * DP * 2) + (c >> 3) * (TC_ROWS * 128) + rr * 128 + (((c & 7) ^ (rr & 7)) * 16);
}

template <typename T, int DP>
__global__ void __launch_bounds__(TC_THREADS, 1)
paged_chunk_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV,
                   const __grid_constant__ TcArgs t) {
    constexpr int ST = tc_stages<DP>();
    constexpr int TILE = tc_tile_bytes<DP>();
    constexpr int HALVES = DP / 64;                    // 128-byte column blocks
    extern __shared__ __align__(1024) unsigned char smem_raw[];
    // The swizzle needs 1,024-byte alignment, which the array's alignment gives (there is
    // no room to round up to it); should it ever not, the call says so.
    if ((smem_u32(smem_raw) & 1023u) != 0) {
        if (threadIdx.x == 0) atomicOr(t.a.status, HMM_STATUS_TIMEOUT);
        return;
    }
    unsigned char* Qs = smem_raw;                      // [tile][half][128 rows][128 B], swizzled
    unsigned char* Rs = Qs + tc_q_bytes<DP>();         // ring: [stage][half][128 keys][128 B]
    TcCtrl* ctl = reinterpret_cast<TcCtrl*>(Rs + ST * TILE);
    const AttnArgs& a = t.a;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

    // ---- this CTA's unit
    {
        int64_t run = 0;
        bool found = false;
        for (int s0 = 0; s0 < a.b.n_seq; s0 += TC_THREADS) {
            const int s = s0 + threadIdx.x;
            int64_t v = 0;
            Seq mine{0, 0, 0, false};
            if (s < a.b.n_seq) {
                mine = load_seq(a.b, a.max_kv, s, a.status);
                v = tc_load(t, mine).blocks;
            }
            int64_t incl = v;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int64_t u = __shfl_up_sync(0xffffffffu, incl, o);
                if (lane >= o) incl += u;
            }
            if (lane == 31) ctl->scan[warp] = incl;
            __syncthreads();
            int64_t sum = 0;
#pragma unroll
            for (int w = 0; w < TC_WARPS; ++w) {
                if (w < warp) incl += ctl->scan[w];
                sum += ctl->scan[w];
            }
            incl += run;
            if (incl - v <= (int64_t)blockIdx.x && (int64_t)blockIdx.x < incl) {
                ctl->seq = s;
                ctl->own = mine;
                ctl->pre = incl - v;
            }
            run += sum;
            found = run > (int64_t)blockIdx.x;
            __syncthreads();
            if (found) break;
        }
        if (!found) return;
    }
    const int s = ctl->seq;
    const Seq q = ctl->own;
    const TcLoad ld = tc_load(t, q);
    const int unit = (int)(blockIdx.x - ctl->pre);
    // a sequence's last rows see the most keys: they go first, so that the
    // short blocks fill the end
    const int kvh = unit % a.hk, rb = ld.row_blocks - 1 - unit / a.hk;
    const int row0 = rb * TC_CTA_ROWS;
    const int rows = (int)min((int64_t)TC_CTA_ROWS, (int64_t)q.n_new * a.group - row0);
    const Span sp = tile_span(a, q, row0, row0 + rows);
    const int sink_tiles = (sp.sink + TC_KEYS - 1) / TC_KEYS;
    const int first = max(sp.lo / TC_KEYS, sink_tiles);
    auto tiles_to = [&](int hi) { return sink_tiles + max(0, (hi + TC_KEYS - 1) / TC_KEYS - first); };
    auto key0_of = [&](int j) { return (j < sink_tiles ? j : first + j - sink_tiles) * TC_KEYS; };
    // tiles with keys that no row sees beside some that are seen
    auto mends = [&](int key0) {
        return !(key0 >= sp.lo && key0 + TC_KEYS <= sp.hi) && key0 + TC_KEYS > sp.sink;
    };
    // key tiles of each row tile: a prefix of the CTA's
    int n_of[TC_TILES];
#pragma unroll
    for (int w = 0; w < TC_TILES; ++w) {
        const int r0 = row0 + w * TC_ROWS, r1 = min(row0 + rows, r0 + TC_ROWS);
        n_of[w] = r0 < r1 ? tiles_to(tile_span(a, q, r0, r1).hi) : 0;
    }
    const int n = max(n_of[0], n_of[1]);
    volatile int* abort = &ctl->abort;

    if (threadIdx.x == 0) {
        for (int i = 0; i < ST; ++i) {
            mbar_init(&ctl->full[i], 1);
            mbar_init(&ctl->empty[i], 1);
        }
        for (int w = 0; w < TC_TILES; ++w) {
            mbar_init(&ctl->s_full[w], 1);
            mbar_init(&ctl->p_full[w][0], TC_SOFTMAX_WARPS / 2);
            mbar_init(&ctl->p_full[w][1], TC_SOFTMAX_WARPS / 2);
        }
        mbar_init(&ctl->q_full, TC_SOFTMAX_WARPS);
        mbar_init(&ctl->v_mend, 1);
        mbar_init(&ctl->v_fixed, 1);
        mbar_init(&ctl->o_full, 1);
        mbar_init(&ctl->drain, 1);
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

    // The same setmaxnreg for all warps of a warpgroup; what is outside of the roles runs
    // with the launch's registers again.
    if (warp >= TC_SOFTMAX_WARPS) {
        set_regs_down<TC_REGS_OTHER>();
        if (warp == TC_SOFTMAX_WARPS) {
            // -------------------------------------------------------- producer
            const int br = t.box_rows, subs = TC_KEYS / br;
            if (lane == 0) {
                prefetch_tmap(&tmK);
                prefetch_tmap(&tmV);
            }
            auto lookup = [&](int j, int* page, int* row) {   // lane: box `lane` of tile j
                *page = a.n_pages;                            // out of range: zeros
                *row = 0;
                if (j < n && lane < subs) {
                    const int k0 = key0_of(j) + lane * br;
                    if (k0 < sp.sink || (k0 + br > sp.lo && k0 < sp.hi)) {
                        const int e = page_of(a, s, k0 / a.page_tokens);
                        if (e >= 0) {
                            *page = e;
                            *row = k0 % a.page_tokens;
                        }
                    }
                }
            };
            int page, row, issued = 0;
            bool ok = true;
            lookup(0, &page, &row);
            for (int j = 0; ok && j < n; ++j) {
                int next_page, next_row;
                lookup(j + 1, &next_page, &next_row);
                for (int kv = 0; kv < 2; ++kv) {
                    const int i = 2 * j + kv, st = i % ST;
                    if (!wait_warp(&ctl->empty[st], ((i / ST) & 1) ^ 1, abort, t.wait_ns)) {
                        ok = false;
                        break;
                    }
                    if (lane == 0) mbar_expect_tx(&ctl->full[st], TILE);
                    __syncwarp();
                    issued = i + 1;
                    if (lane < subs) {
                        const uint32_t dst = smem_u32(Rs + st * TILE) + lane * br * 128;
#pragma unroll
                        for (int h = 0; h < HALVES; ++h)
                            tma_load_page(dst + h * (TC_KEYS * 128), kv ? &tmV : &tmK, &ctl->full[st], 64 * h, row,
                                        kvh, page);
                    }
                }
                page = next_page;
                row = next_row;
            }
            if (!ok) {
                if (lane == 0) {
                    atomicExch(&ctl->abort, 1);
                    atomicOr(a.status, HMM_STATUS_TIMEOUT);
                }
                for (int i = max(0, issued - ST); i < issued; ++i)   // copies in flight land first
                    mbar_wait_drain(&ctl->full[i % ST], (i / ST) & 1);
            }
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
            const int nu = __shfl_sync(0xffffffffu, n, 0);
            const int nu_of[2] = {__shfl_sync(0xffffffffu, n_of[0], 0), __shfl_sync(0xffffffffu, n_of[1], 0)};
            auto wait = [&](uint64_t* bar, uint32_t parity) {
                return wait_warp(bar, parity, abort, t.wait_ns);
            };
            auto qk = [&](int w, uint32_t k) {
                const uint32_t ql = qlo + w * (TC_ROWS * DP * 2 / 16), d = tm + 128 * w;
#pragma unroll
                for (int ks = 0; ks < DP / 16; ++ks) {
                    const uint32_t off = ((ks >> 2) * (TC_ROWS * 128) + (ks & 3) * 32) / 16;
                    mma_ss(one, d, ql + off, khi, k + off, khi, id_qk, ks != 0);
                }
                commit_one(one, &ctl->s_full[w]);
            };
            if (nu > 0) {
                int fixed = 0, sv = 1, pv = 0, sk = 2 % ST, pk = 2 / ST;   // stages of V_j, K_j+1 and their phases
                bool ok = wait(&ctl->q_full, 0) && wait(&ctl->full[0], 0);
                if (ok) {
                    tc_fence_after();
#pragma unroll
                    for (int w = 0; w < TC_TILES; ++w)
                        if (nu_of[w] > 0) qk(w, klo);
                    commit_one(one, &ctl->empty[0]);
                }
                for (int j = 0; ok && j < nu; ++j) {
                    const uint32_t v = vlo + sv * (TILE / 16), k = klo + sk * (TILE / 16);
                    if (!(ok = wait(&ctl->full[sv], pv))) break;
                    if (mends(key0_of(j))) {
                        if (lane == 0) mbar_arrive(&ctl->v_mend);
                        if (!(ok = wait(&ctl->v_fixed, fixed++ & 1))) break;
                    }
                    bool k_ready = false;
#pragma unroll
                    for (int w = 0; w < TC_TILES; ++w) {
                        if (j >= nu_of[w]) continue;
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            if (!(ok = wait(&ctl->p_full[w][h], j & 1))) break;
                            tc_fence_after();
#pragma unroll
                            for (int ks = 4 * h; ks < 4 * h + 4; ++ks)
                                mma_ts(one, tm + 256 + DP * w, tm + 128 * w + 8 * ks, v + ks * 128, vhi, id_pv,
                                       j > 0 || ks > 0);
                        }
                        if (!ok) break;
                        if (j + 1 < nu_of[w]) {
                            if (!k_ready && !(ok = wait(&ctl->full[sk], pk))) break;
                            k_ready = true;
                            qk(w, k);
                        }
                    }
                    if (!ok) break;
                    commit_one(one, &ctl->empty[sv]);
                    if (j + 1 < nu) commit_one(one, &ctl->empty[sk]);
                    else commit_one(one, &ctl->o_full);
                    if ((sv += 2) >= ST) { sv -= ST; pv ^= 1; }
                    if ((sk += 2) >= ST) { sk -= ST; pk ^= 1; }
                }
                if (!ok) {
                    if (lane == 0) {
                        atomicExch(&ctl->abort, 1);
                        atomicOr(a.status, HMM_STATUS_TIMEOUT);
                    }
                    commit_one(one, &ctl->drain);    // the MMAs issued end before TMEM is freed
                    mbar_wait_drain(&ctl->drain, 0);
                }
            }
            __syncwarp();
        } else if (warp == TC_SOFTMAX_WARPS + 2) {
            // ------------------------------------------------ V's unseen rows
            // V rows that no row of the CTA sees, in boxes that were read, become zeros:
            // a weight of zero times what a slot of nobody holds is only zero then.
            // The MMA lane says when such a tile has arrived, and waits: this warp, which
            // skips the others, could not tell a stage's phases apart.
            int mended = 0;
            for (int j = 0; j < n; ++j) {
                const int key0 = key0_of(j), st = (2 * j + 1) % ST;
                if (!mends(key0)) continue;
                if (!wait_warp(&ctl->v_mend, mended++ & 1, abort, t.wait_ns)) break;
                for (int r = lane; r < TC_KEYS; r += 32) {
                    const int key = key0 + r, k0 = key - r % t.box_rows;
                    if (!span_has(sp, key) && (k0 < sp.sink || (k0 + t.box_rows > sp.lo && k0 < sp.hi))) {
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
        }
        tc_fence_before();
        roles_done();
        set_regs_up<TC_REGS_LAUNCH>();   // the softmax warps have given theirs back
    } else {
        // --------------------------------------------------------- softmax
        set_regs_up<TC_REGS_SOFTMAX>();
        // Two threads share a row: part p has the scores of keys [32 p, 32 p + 32) and
        // [64 + 32 p, 96 + 32 p) of a tile, and half of the row's results.  Two warps per
        // row tile on each scheduler keep the special-function unit busy where one, with
        // the maxima and the conversions between, leaves it idle half of the time.
        {
            // q rows, swizzled
            constexpr int CH = DP / 8;
            const uint32_t q0 = smem_u32(Qs);
#pragma unroll
            for (int i = 0; i < TC_CTA_ROWS * CH / TC_SOFTMAX; ++i) {
                const int at = i * TC_SOFTMAX + threadIdx.x, r = at / CH, c = at % CH;
                const bool real = r < rows && c * 8 < a.D;
                const int tok = a.by_group(row0 + (real ? r : 0)), head = row0 + (real ? r : 0) - tok * a.group;
                cp16(q0 + q_at<DP>(r, c),
                     a.q + (int64_t)(q.begin + tok) * a.q_token + (int64_t)(kvh * a.group + head) * a.q_head + (real ? 16 * c : 0),
                     real);
            }
            cp_commit();
            cp_wait<0>();
            if (a.scale < 0.0f) {   // turned signs: the largest score is the largest product
#pragma unroll 1
                for (int i = 0; i < TC_CTA_ROWS * CH / TC_SOFTMAX; ++i) {
                    const int at = i * TC_SOFTMAX + threadIdx.x;
                    uint4* x = reinterpret_cast<uint4*>(Qs + q_at<DP>(at / CH, at % CH));
                    *x = make_uint4(x->x ^ 0x80008000u, x->y ^ 0x80008000u, x->z ^ 0x80008000u, x->w ^ 0x80008000u);
                }
            }
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(&ctl->q_full);
        }
        const int w = warp >> 3, part = (warp >> 2) & 1;
        const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
        const uint32_t ts = tmem + 128 * w + lanes, to = tmem + 256 + DP * w + part * (DP / 2) + lanes;
        const int r = w * TC_ROWS + (warp & 3) * 32 + lane;   // row of the CTA
        const int wr0 = r - lane;                              // the warp's rows: [wr0, wr1)
        const int wr1 = min(rows, wr0 + 32);
        const int pair = 2 + w * 4 + (warp & 3);               // barrier of the two warps of these rows
        const int pos = row_pos(a, q, row0 + min(r, rows - 1));
        const int pos_first = row_pos(a, q, row0 + min(wr0, rows - 1));
        const int pos_last = row_pos(a, q, row0 + max(wr1, 1) - 1);
        const float sc = fabsf(a.scale_log2);
        const uint64_t sc2 = pack_f2(sc, sc);
        float m = -INFINITY;
        uint64_t l2[2] = {pack_f2(0.0f, 0.0f), pack_f2(0.0f, 0.0f)};
        bool ok = true, fine = true;
        const int nw = n_of[w];
        for (int j = 0; j < nw; ++j) {
            // (a warp that gave up keeps the pair's count of barriers: its partner may not
            // have, or at another tile)
            if (ok) ok = wait_warp(&ctl->s_full[w], j & 1, abort, t.wait_ns);
            if (!ok) {
                pair_sync(pair);
                continue;
            }
            tc_fence_after();
            uint32_t v[64];
            tmem_ld_x32(ts + 32 * part, v);
            tmem_ld_x32(ts + 64 + 32 * part, v + 32);
            tmem_wait_ld();
            const int key0 = key0_of(j);
            if (!(key0 + TC_KEYS <= q.kv && (!a.causal || key0 + TC_KEYS - 1 <= pos_first) &&
                  (a.window <= 0 || key0 > pos_last - a.window || key0 + TC_KEYS <= a.sinks))) {
                const int at = key0 + 32 * part;
                const int hi = (a.causal ? min(q.kv, pos + 1) : q.kv) - at;
                const int lo = a.window > 0 ? max(0, pos - a.window + 1) - at : -TC_KEYS;
                const int sink = a.window > 0 ? a.sinks - at : 0;
#pragma unroll
                for (int i = 0; i < 64; ++i) {
                    const int c = i < 32 ? i : i + 32;
                    if (c >= hi || (c < lo && c >= sink)) v[i] = 0xff800000u;
                }
            }
            // The first half's weights with the maximum so far, while this tile's is found:
            // that is right unless the row grew by more than TC_GROWTH, which is rare.
            uint32_t p[16];
            uint64_t sum;
            // NaN and +inf show in the maximum: such a row is computed again at the end.
            float top = weights<T, true>(v, sc2, m, sc, p, &sum);
            ctl->top[part][r] = top;   // read before the partner's weights, and so before the next tile
            pair_sync(pair);
            top = max3(top, ctl->top[part ^ 1][r], top);
            fine = fine && top < INFINITY;
            const bool grow = (top - m) * sc > TC_GROWTH;
            if (__any_sync(0xffffffffu, grow)) {
                const float al = grow ? ex2((m - top) * sc) : 1.0f;
                if (grow) m = top;
                const uint64_t al2 = pack_f2(al, al);
                l2[0] = fma_f2(l2[0], al2, pack_f2(0.0f, 0.0f));
                l2[1] = fma_f2(l2[1], al2, pack_f2(0.0f, 0.0f));
                if (j > 0) {
#pragma unroll 1
                    for (int c = 0; c < DP / 2; c += 16) {
                        uint32_t o[16];
                        tmem_ld_x16(to + c, o);
                        tmem_wait_ld();
#pragma unroll
                        for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * al);
                        tmem_st_x16(to + c, o);
                    }
                }
                weights<T, false>(v, sc2, m, sc, p, &sum);
            }
            // the first half's product starts while the second half is in the exponentials
            tmem_st_x16(ts + 16 * part, p);
            l2[0] = add_f2(l2[0], sum);
            tmem_wait_st();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&ctl->p_full[w][0]);
            weights<T, false>(v + 32, sc2, m, sc, p, &sum);
            tmem_st_x16(ts + 32 + 16 * part, p);
            l2[1] = add_f2(l2[1], sum);
            tmem_wait_st();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&ctl->p_full[w][1]);
        }
        // ---- the rows' results
        if (ok && n > 0) ok = wait_warp(&ctl->o_full, 0, abort, t.wait_ns);
        float l, lb;
        unpack_f2(add_f2(l2[0], l2[1]), l, lb);
        ctl->top[part][r] = l + lb;
        if (!ok && lane == 0) {
            atomicExch(&ctl->abort, 1);
            atomicOr(a.status, HMM_STATUS_TIMEOUT);
        }
        pair_sync(pair);
        // (after a wait that ran out, too: every warp passes the same barriers, and what it
        // writes, in its own rows, is as invalid as the call says)
        {
            tc_fence_after();
            l = ctl->top[0][r] + ctl->top[1][r];
            const bool live = r < rows;
            const int tok = a.by_group(row0 + (live ? r : 0)), head = row0 + (live ? r : 0) - tok * a.group;
            const int64_t orow = (int64_t)(q.begin + tok) * a.hq + kvh * a.group + head;
            const float inv = l == 0.0f ? 0.0f : 1.0f / l;
            fine = fine && l == l;
            // through shared memory (every product is complete), rows 16 bytes apart in
            // their banks, so that whole rows go out at once
            constexpr int OROW = DP * 2 + 16;
            unsigned char* os = smem_raw + r * OROW + part * DP;
#pragma unroll
            for (int c = 0; c < DP / 2; c += 16) {
                uint32_t o[16];
                if (nw > 0) {
                    tmem_ld_x16(to + c, o);
                    tmem_wait_ld();
                }
#pragma unroll
                for (int i = 0; i < 16; i += 8) {
                    float f[8];
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        f[e] = nw > 0 && l != 0.0f ? __uint_as_float(o[i + e]) * inv : 0.0f;
                        if (part * (DP / 2) + c + i < a.D) fine = fine && fabsf(f[e]) < INFINITY;
                    }
                    *reinterpret_cast<uint4*>(os + 2 * (c + i)) =
                        make_uint4(pack2<T>(f[0], f[1]), pack2<T>(f[2], f[3]), pack2<T>(f[4], f[5]),
                                   pack2<T>(f[6], f[7]));
                }
            }
            pair_sync(pair);
            constexpr int CH = DP / 8;                 // 16-byte pieces of a row
            const int c = lane % CH;
#pragma unroll
            for (int i = 0; i < 16; i += 32 / CH) {    // this warp's half of the pair's rows
                const int rr = 16 * part + i + lane / CH;
                const int64_t to_row = __shfl_sync(0xffffffffu, orow, rr);
                if (wr0 + rr < rows && c * 8 < a.D)
                    *reinterpret_cast<uint4*>(a.out + 2 * (to_row * a.D + 8 * c)) =
                        *reinterpret_cast<const uint4*>(smem_raw + (wr0 + rr) * OROW + 16 * c);
            }
            if (live && a.lse && part == 0)
                a.lse[orow] = l == 0.0f ? -INFINITY : ((m == -INFINITY ? 0.0f : m * sc) + log2f(l)) * LN2;
            const unsigned again = __ballot_sync(0xffffffffu, live && !fine);
            if (lane == 0) ctl->again[warp] = again;
        }
        set_regs_down<TC_REGS_LAUNCH>();
        tc_fence_before();
        roles_done();
    }
    tc_fence_after();
    if (warp == TC_SOFTMAX_WARPS + 1) tmem_dealloc(tmem, 512);
    if (warp < TC_CTA_ROWS / 32) {   // rows [32 warp, 32 warp + 32)
        const int at = (warp >> 2) * 8 + (warp & 3);
        unsigned again = *abort ? 0u : ctl->again[at] | ctl->again[at + 4];
        while (again) {
            const int i = __ffs(again) - 1;
            again &= again - 1;
            attn_row_exact<T>(a, s, q, kvh, row0 + warp * 32 + i);
        }
    }
}

PFN_cuTensorMapEncodeTiled_v12000 encode_fn() {
    static PFN_cuTensorMapEncodeTiled_v12000 fn = nullptr;
    static std::once_flag once;
    std::call_once(once, [] {
        void* p = nullptr;
        cudaDriverEntryPointQueryResult r;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &r) == cudaSuccess &&
            r == cudaDriverEntryPointSuccess)
            fn = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(p);
    });
    return fn;
}

template <typename T, int DP>
hmm_status_t launch_chunk(const TcArgs& t, const CUtensorMap& k, const CUtensorMap& v, unsigned grid,
                          cudaStream_t st) {
    static std::atomic<uint64_t> done{0};
    const hmm_status_t s = allow_smem(paged_chunk_kernel<T, DP>, tc_smem<DP>(), &done);
    if (s != HMM_OK) return s;
    paged_chunk_kernel<T, DP><<<grid, TC_THREADS, tc_smem<DP>(), st>>>(k, v, t);
    return check_launch("paged_chunk_kernel");
}

}  // namespace

hmm_status_t make_page_map(CUtensorMap* m, const AttnArgs& a, const Pages& p, int box_rows) {
    auto fn = encode_fn();
    if (!fn) return set_error(HMM_ERR_CUDA, "cuTensorMapEncodeTiled is unavailable");
    cuuint64_t dims[4] = {(cuuint64_t)a.D, (cuuint64_t)a.page_tokens, (cuuint64_t)a.hk, (cuuint64_t)a.n_pages};
    cuuint64_t strides[3] = {(cuuint64_t)p.token, (cuuint64_t)p.head, (cuuint64_t)p.page};
    for (int i = 0; i < 3; ++i)
        if (dims[i + 1] == 1) strides[i] = 16;   // never stepped over
    cuuint32_t box[4] = {64, (cuuint32_t)box_rows, 1, 1};
    cuuint32_t ones[4] = {1, 1, 1, 1};
    const CUresult r = fn(m, CU_TENSOR_MAP_DATA_TYPE_UINT16, 4, p.base, dims, strides, box, ones,
                          CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                          CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return set_error(HMM_ERR_CUDA, "cuTensorMapEncodeTiled failed (%d)", (int)r);
    return HMM_OK;
}

bool chunk_applies(const AttnArgs& a) {
    return a.D <= 128 && box_rows_of(a.page_tokens, TC_KEYS) >= 8;
}

hmm_status_t run_chunk(const AttnArgs& a, bool bf16, int min_rows, cudaStream_t st) {
    TcArgs t{a, min_rows, box_rows_of(a.page_tokens, TC_KEYS), wait_limit_ns()};
    CUtensorMap k, v;
    hmm_status_t s = make_page_map(&k, a, a.k, t.box_rows);
    if (s != HMM_OK) return s;
    s = make_page_map(&v, a, a.v, t.box_rows);
    if (s != HMM_OK) return s;
    // every sequence's rows in blocks: one more than its share of the tokens at most
    const int64_t most = ((int64_t)a.b.n_tokens * a.group / TC_CTA_ROWS + a.b.n_seq) * a.hk;
    HMM_REQUIRE(most < (int64_t(1) << 31), "n_tokens * n_heads is too large for one call");
    const unsigned grid = (unsigned)most;
    if (a.D <= 64)
        return bf16 ? launch_chunk<__nv_bfloat16, 64>(t, k, v, grid, st) : launch_chunk<__half, 64>(t, k, v, grid, st);
    return bf16 ? launch_chunk<__nv_bfloat16, 128>(t, k, v, grid, st) : launch_chunk<__half, 128>(t, k, v, grid, st);
}

}  // namespace serve
}  // namespace hmm
