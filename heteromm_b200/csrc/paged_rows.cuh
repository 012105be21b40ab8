// paged_rows.cuh — attention of few rows (decoding, drafted tokens) over a paged cache of
// 16-bit values or in 8 bits, the join of what several CTAs summed, and the choice between
// this kernel and the one for chunks.
//
// paged_rows_kernel.  A unit is (sequence, KV head, 16 rows): rows are (new
// token, query head of the group), so grouped heads read their keys once.  With
// few rows the cache has to be read for next to no arithmetic and HBM bounds it;
// the design keeps reads in flight:
//   - all units' key tiles form one list, cut into as many equal pieces as CTAs
//     fit the GPU (ragged lengths balance by themselves); a CTA finds its piece
//     from the lengths on the device, so no host value goes stale;
//   - each warp owns 16 keys of a tile (of a cache in 8 bits 32: as many bytes) and its own ring of
//     TMA stages, with no barrier between warps: a box per 128 bytes of a page's rows, issued by
//     one elected lane (by as many lanes as boxes the hardware took one lane after the other: of a
//     tile's 2,500 clocks 950, and 640 so), its page looked up one stage ahead and checked when it is
//     used, zeros for the boxes that no row of the tile sees.  With 16-byte cp.async instead the
//     L1 cache held the bytes in flight (478 us, 8 bits 361);
//   - scores and the product with V on mma.sync (m16n8k16, fp32 sums), the
//     running maximum and sum in fp32 per warp, warps joined once per piece;
//   - a unit that several CTAs share leaves (maximum, sum, unnormalised rows) per
//     piece in the workspace, and paged_join_kernel adds the pieces in order.
// Measured: 64 sequences of up to 16,384 tokens, one new token each, 32 query and 8 KV
// heads of 128: 347-351 us, 6.3 TB/s (cp.async: 478); one token over 777: 12.5 us, of
// which 2.5 the join, over 4,000 18.8 us.  The same decode batch in e4m3: 248 us, 4.6 TB/s, where
// HBM would allow 173: conversions, scores and softmax are 4,000 clocks of latency a tile for a
// warp, and twelve warps an SM hide a part of them.
#pragma once

#include <algorithm>

#include "paged_attn.cuh"
#include "paged_attn_tc.cuh"
#include "paged_code_tile.cuh"

namespace hmm {
namespace serve {
using namespace sm100;

constexpr int RW_WARPS = 4;
constexpr int RW_THREADS = 32 * RW_WARPS;
constexpr int RW_ROWS = 16;
// Keys of a warp's tile, and of a CTA's: as many bytes of either cache, so that what a tile costs
// beside them is the same.
template <int C>
__host__ __device__ constexpr int rows_keys() { return C == CODEC_NONE ? 16 : 32; }
template <int C>
__host__ __device__ constexpr int rows_tile() { return RW_WARPS * rows_keys<C>(); }

struct RowsWork {
    int4* joint;      // [ctas][2] unit begun in the CTA and ended in another: sequence, head, row tile,
                      // pieces (0: none); the sequence's begin, n_new, kv
    float* part;      // [ctas][2][RW_ROWS * (DP + 2)]: rows, then maxima, then sums
};

struct RowsArgs {
    AttnArgs a;
    RowsWork w;
    int max_rows;     // sequences of more rows are another kernel's
    int box_rows;     // rows of a TMA box: a power of two that divides page_tokens
    uint64_t wait_ns; // limit of every bounded wait
};

// Rows of a sequence that are this kernel's where the chunk kernel takes its caches too (one row
// tile or two; at run_kernels).
template <int C>
__host__ __device__ constexpr int rows_most() { return C == CODEC_NONE ? RW_ROWS : 2 * RW_ROWS; }

// CTAs of an SM at D <= 128 (64: four; 256: one): two with three stages a warp keep the bytes in flight
// that HBM wants and start soonest; with three of two stages more instructions are in flight, and
// more units' starts and ends.  In 8 bits the decode batch takes 247 us with three and 293 with two,
// 16-bit sequences of 1,000 behind a shared prefix 111 and 123; one token over 777 13.9 and 12.8.
template <int DP, int C>
__host__ __device__ constexpr int rows_ctas_per_sm(bool shared) {
    return DP == 64 ? 4 : DP == 128 ? (C == CODEC_NONE && !shared ? 2 : 3) : 1;
}
template <int DP>
__host__ __device__ constexpr int rows_stages(int ctas) { return DP == 128 && ctas == 3 ? 2 : 3; }

// A stage of a warp: K, then V; in 8 bits their scale bytes lie behind all warps' rings.
template <int DP, int C>
__host__ __device__ constexpr int rows_stage() { return 2 * rows_keys<C>() * DP * (C == CODEC_NONE ? 2 : 1); }
template <int DP, int C>
__host__ __device__ constexpr int rows_scales() { return C == CODEC_NONE ? 0 : 2 * rows_keys<C>() * DP / Q_GROUP; }
template <int DP, int C, int CTAS>
constexpr size_t rows_smem() {
    return 1024 + (size_t)RW_WARPS * rows_stages<DP>(CTAS) * (rows_stage<DP, C>() + rows_scales<DP, C>());
}

__device__ __forceinline__ void ldm4(uint32_t* r, uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr));
}
__device__ __forceinline__ void ldm4t(uint32_t* r, uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr));
}

template <typename T>
__device__ __forceinline__ void mma16816(float* d, const uint32_t* a, uint32_t b0, uint32_t b1);
template <>
__device__ __forceinline__ void mma16816<__nv_bfloat16>(float* d, const uint32_t* a, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <>
__device__ __forceinline__ void mma16816<__half>(float* d, const uint32_t* a, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// Units and key tiles of a sequence.  `tiles` is the same for each of its
// units, an upper bound of what a unit's rows see.
struct Load {
    int units, tiles, row_tiles;
};

template <int C>
__device__ __forceinline__ Load seq_load(const RowsArgs& r, const Seq& q) {
    constexpr int TILE = rows_tile<C>();
    const int64_t rows = (int64_t)q.n_new * r.a.group;
    Load x{0, 0, 0};
    if (rows == 0 || rows > r.max_rows) return x;
    x.row_tiles = (int)((rows + RW_ROWS - 1) / RW_ROWS);
    x.units = x.row_tiles * r.a.hk;
    int64_t t = ((int64_t)q.kv + TILE - 1) / TILE - q.lo / TILE;
    if (r.a.window > 0) {
        const int64_t near = ((int64_t)r.a.window + RW_ROWS + TILE - 1) / TILE + 1;
        t = min(t, near + ((int64_t)r.a.sinks + TILE - 1) / TILE);
    }
    x.tiles = (int)max(t, (int64_t)1);   // a row that sees nothing is written too
    return x;
}

// Inclusive scan over the block's threads.
__device__ __forceinline__ int64_t scan_incl(int64_t v, int64_t* wt, int64_t* total) {
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int64_t t = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= o) v += t;
    }
    if (lane == 31) wt[w] = v;
    __syncthreads();
    int64_t add = 0, sum = 0;
#pragma unroll
    for (int i = 0; i < RW_WARPS; ++i) {
        if (i < w) add += wt[i];
        sum += wt[i];
    }
    __syncthreads();
    *total = sum;
    return v + add;
}

// (apart from the kernel's code, which streams)
template <typename T, int C>
__device__ __noinline__ void rows_exact(const AttnArgs& a, const Seq& q, int kvh, int row0, unsigned rows) {
    attn_rows_exact<T, C, 1>(a, q, kvh, row0, rows);
}

template <typename T, int DP, int C, int CTAS>
__global__ void __launch_bounds__(RW_THREADS, CTAS)
paged_rows_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV,
                  const __grid_constant__ RowsArgs r) {
    extern __shared__ __align__(1024) unsigned char smem_raw[];
    unsigned char* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
    constexpr int RW_STAGES = rows_stages<DP>(CTAS);
    __shared__ uint64_t full[RW_WARPS][RW_STAGES];
    __shared__ int64_t wt[RW_WARPS];
    __shared__ int64_t sh_pre;
    __shared__ int sh_seq, again, any_again, abort;
    __shared__ uint4 qs[C != CODEC_NONE ? DP * 2 : 1];   // in 8 bits: the unit's queries [step][lane]
    constexpr bool QUANT = C != CODEC_NONE;
    constexpr int KEYS = rows_keys<C>(), TILE = rows_tile<C>();
    // A box is 128 bytes of a row (64 values, or 128 codes; 64 codes at D = 64), swizzled over as
    // many bytes.
    constexpr int ROW = QUANT && DP == 64 ? 64 : 128, HALVES = QUANT ? (DP + 127) / 128 : DP / 64;
    constexpr int BLOCK = KEYS * ROW;
    constexpr int STAGE = rows_stage<DP, C>(), SCALES = rows_scales<DP, C>();
    constexpr int MR = DP + 4;                         // joining rows: 4 banks apart
    using M = std::conditional_t<QUANT, __half, T>;    // the products' type
    // log2 of what weights are held by: the largest is 2^14 in fp16, whose range ends at 2^-25
    // (a key 18 nats below the largest had no weight at all, and a long tail of them a share
    // of the result).  It cancels against the sum, and lse takes it back with the maximum.
    constexpr float UP = std::is_same<M, __half>::value ? 14.0f : 0.0f;
    const AttnArgs& a = r.a;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    // (Parts are the kernel before's, which this one is launched ahead of; so the next may not start
    // before either.)
    if (a.b.shared) asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

    if (threadIdx.x == 0) {
        for (int w = 0; w < RW_WARPS; ++w)
            for (int i = 0; i < RW_STAGES; ++i) mbar_init(&full[w][i], 1);
        abort = any_again = 0;
        fence_barrier_init();
    }
    // ---- this CTA's piece of the list of all units' tiles
    int64_t total = 0, own = 0;
    each_seq(a.b, a.max_kv, threadIdx.x, RW_THREADS, a.status, [&](const Seq& q) {
        const Load x = seq_load<C>(r, q);
        own += (int64_t)x.units * x.tiles;
    });
    scan_incl(own, wt, &total);
    const int64_t share = max((int64_t)1, (total + gridDim.x - 1) / gridDim.x);
    int64_t cur = blockIdx.x * share;
    const int64_t end = min(total, cur + share);
    if (threadIdx.x == 0) r.w.joint[2 * blockIdx.x] = make_int4(0, 0, 0, 0);
    if (cur >= end) return;
    {
        int64_t run = 0;
        for (int s0 = 0; s0 < a.b.n_seq; s0 += RW_THREADS) {
            const int s = s0 + threadIdx.x;
            int64_t v = 0, sum;
            if (s < a.b.n_seq) {
                const Load x = seq_load<C>(r, load_seq(a.b, a.max_kv, s, a.status));
                v = (int64_t)x.units * x.tiles;
            }
            const int64_t incl = scan_incl(v, wt, &sum) + run;
            if (incl - v <= cur && cur < incl) {
                sh_seq = s;
                sh_pre = incl - v;
            }
            run += sum;
            if (run > cur) break;
        }
        __syncthreads();
    }
    int s = sh_seq;
    int64_t pre = sh_pre;                              // tiles before sequence s
    Seq q = load_seq(a.b, a.max_kv, s, a.status);
    Load ld = seq_load<C>(r, q);

    unsigned char* ring_p = smem + warp * RW_STAGES * STAGE;
    const uint32_t ring = smem_u32(ring_p);
    unsigned char* scales_p = smem + RW_WARPS * RW_STAGES * STAGE + warp * RW_STAGES * SCALES;
    const int per = QUANT ? a.quant.per_token : 0;     // scale bytes of a token
    // boxes of the warp's keys, one after the other: lane: [sub * box_rows, +box_rows)
    const int subs = KEYS / r.box_rows, sub = lane % subs;
    uint32_t done = 0;                                 // tiles that the ring has seen
    bool dead = false;                                 // a wait gave up: no more copies
    while (cur < end) {
        while (cur >= pre + (int64_t)ld.units * ld.tiles) {
            pre += (int64_t)ld.units * ld.tiles;
            q = load_seq(a.b, a.max_kv, ++s, a.status);
            ld = seq_load<C>(r, q);
        }
        const int unit = (int)((cur - pre) / ld.tiles);
        const int t0 = (int)(cur - pre - (int64_t)unit * ld.tiles);
        const int t1 = (int)min((int64_t)ld.tiles, t0 + (end - cur));
        const int kvh = unit / ld.row_tiles, rt = unit - kvh * ld.row_tiles;
        const int row0 = rt * RW_ROWS;
        const int rows = (int)min((int64_t)RW_ROWS, (int64_t)q.n_new * a.group - row0);
        const Span sp = tile_span(a, q, row0, row0 + rows);
        const int sink_tiles = (sp.sink + TILE - 1) / TILE;
        const int first = max(sp.lo / TILE, sink_tiles);
        const int n_tiles = sink_tiles + max(0, (sp.hi + TILE - 1) / TILE - first);
        const int n = min(t1, n_tiles) - t0;           // tiles of this piece, <= 0: none

        auto key0_of = [&](int i) {                    // first key of this warp's part of tile t0 + i
            const int t = t0 + i;
            return (t < sink_tiles ? t : first + t - sink_tiles) * TILE + warp * KEYS;
        };
        const ScaleCopy scale_from = QUANT ? scale_copy(a, kvh, r.box_rows, SCALES / 2) : ScaleCopy{};
        // This lane's box rows of the next tile: the table's entry, looked at when it is used (a check
        // here would wait for it, 1,000 clocks a tile), and the row in its page; -1: none are seen.
        int entry = 0, row = -1;
        auto lookup = [&](int i) {
            row = -1;
            if (i < n) {
                const int k0 = key0_of(i) + sub * r.box_rows;
                if (k0 < sp.sink || (k0 + r.box_rows > sp.lo && k0 < sp.hi)) {
                    const int lp = a.by_page(k0);
                    entry = __ldg(a.b.table + (int64_t)q.row * a.b.pages_per_seq + lp);
                    row = k0 - lp * a.page_tokens;
                }
            }
        };
        auto page_now = [&] {                          // out of range: zeros
            if (row < 0) return a.n_pages;
            if (entry >= 0 && entry < a.n_pages) return entry;
            atomicOr(a.status, HMM_STATUS_PAGE_BOUNDS);
            return a.n_pages;
        };
        auto issue = [&](int i) {                      // copies of tile i, whose lookup is in page / row
            if (i < n && !dead) {
                const int page = page_now();
                const uint32_t st = (done + i) % RW_STAGES;
                if (lane == 0) mbar_expect_tx(&full[warp][st], STAGE);
                __syncwarp();
                uint32_t d = ring + st * STAGE;
                const uint32_t one = elect_one();
                for (int x = 0; x < subs; ++x, d += r.box_rows * ROW) {
                    const int pg = __shfl_sync(0xffffffffu, page, x), rw = max(0, __shfl_sync(0xffffffffu, row, x));
                    if (one) {
#pragma unroll
                        for (int b = 0; b < HALVES; ++b) {
                            tma_load_page(d + b * BLOCK, &tmK, &full[warp][st], b * (QUANT ? 128 : 64), rw, kvh, pg);
                            tma_load_page(d + (HALVES + b) * BLOCK, &tmV, &full[warp][st], b * (QUANT ? 128 : 64), rw, kvh, pg);
                        }
                    }
                }
                if (QUANT)
                    code_copy_scales(a, scale_from, page, row, smem_u32(scales_p + st * SCALES));
            }
            if (QUANT) cp_commit();                    // (a tile that is not there is an empty group)
        };

        // q fragments: rows lane / 4 and lane / 4 + 8
        uint32_t qf[DP / 16][4];
        int pos[2];
        float factor[2] = {a.scale_log2, a.scale_log2};
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int row = lane / 4 + 8 * h;
            const bool real = row < rows;
            const int at = row0 + (real ? row : 0);
            pos[h] = real ? row_pos(a, q, at) : -1;
            const unsigned char* src = a.q + (int64_t)(q.begin + at / a.group) * a.q_token +
                                       (int64_t)(kvh * a.group + at % a.group) * a.q_head;
            if constexpr (QUANT) {
                factor[h] *= code_queries<T, DP>(real ? src : nullptr, a.D, h, qf);
            } else {
#pragma unroll
                for (int k = 0; k < DP / 16; ++k)
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        const int d = k * 16 + j * 8 + (lane & 3) * 2;
                        qf[k][h + 2 * j] = real && d < a.D ? __ldg(reinterpret_cast<const uint32_t*>(src + 2 * d)) : 0u;
                    }
            }
        }
        if constexpr (QUANT) {
#pragma unroll
            for (int k = 0; k < DP / 16; ++k)
                if (k % RW_WARPS == warp) qs[k * 32 + lane] = make_uint4(qf[k][0], qf[k][1], qf[k][2], qf[k][3]);
            __syncthreads();
        }
#pragma unroll
        for (int i = 0; i < RW_STAGES - 1; ++i) {
            lookup(i);
            issue(i);
        }
        lookup(RW_STAGES - 1);

        float o[DP / 8][4];
        float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f};
#pragma unroll
        for (int i = 0; i < DP / 8; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) o[i][j] = 0.0f;

        for (int i = 0; i < n; ++i) {
            if (QUANT) {
                cp_wait<RW_STAGES - 2>();              // a lane's own copies of scale bytes,
                __syncwarp();                          // and the other lanes', which it reads
            }
            if (!dead) {
                const uint32_t at = done + i;
                dead = !__all_sync(0xffffffffu, mbar_wait_bounded(&full[warp][at % RW_STAGES],
                                                                  (at / RW_STAGES) & 1, &abort, r.wait_ns));
                if (dead) {
                    if (lane == 0) {
                        atomicExch(&abort, 1);
                        atomicOr(a.status, HMM_STATUS_TIMEOUT);
                    }
                    for (int k = i; k < min(n, i + RW_STAGES - 1); ++k)   // copies in flight land first
                        mbar_wait_drain(&full[warp][(done + k) % RW_STAGES], ((done + k) / RW_STAGES) & 1);
                }
            }
            issue(i + RW_STAGES - 1);                  // into the stage that tile i - 1 left
            lookup(i + RW_STAGES);
            const uint32_t so = ((done + i) % RW_STAGES) * STAGE;
            const int key0 = key0_of(i);
            if (!(key0 >= sp.lo && key0 + KEYS <= sp.hi) && key0 + KEYS > sp.sink) {
                // V rows that no row of the unit sees, beside some that are seen, become
                // zeros: a weight of zero times what a slot of nobody holds is only zero then
                if (lane < KEYS && !span_has(sp, key0 + lane)) {
#pragma unroll
                    for (int c = 0; c < HALVES * (ROW / 16); ++c)
                        *reinterpret_cast<uint4*>(ring_p + so + (HALVES + c / (ROW / 16)) * BLOCK + lane * ROW +
                                                  c % (ROW / 16) * 16) = make_uint4(0u, 0u, 0u, 0u);
                    // (a slot of nobody may have a scale byte of 255, which would make NaN of a zero)
                    for (int g = 0; g < per; ++g) scales_p[so / STAGE * SCALES + SCALES / 2 + lane * per + g] = 127;
                }
                fence_proxy_async_smem();              // before the stage's next copies
                __syncwarp();
            }
            constexpr int NB = KEYS / 8;               // blocks of 8 keys
            float sc[NB][4] = {};
            const int mi = lane >> 3, ml = lane & 7;
            const uint32_t kt = ring + so, vt = kt + STAGE / 2;
            const unsigned char* scales = scales_p + so / STAGE * SCALES;
            if constexpr (QUANT) {
                code_scores<DP, C>(ring_p + so, scales, per, qs, sc);
            } else {
#pragma unroll
                for (int k = 0; k < DP / 16; ++k) {
                    uint32_t b[4];
                    const int row = ml + (mi >> 1) * 8, c = 2 * k + (mi & 1);
                    ldm4(b, kt + (c >> 3) * BLOCK + row * 128 + (((c & 7) ^ (row & 7)) * 16));
                    mma16816<T>(sc[0], qf[k], b[0], b[1]);
                    mma16816<T>(sc[1], qf[k], b[2], b[3]);
                }
            }
            const bool all = key0 + KEYS <= q.kv && (!a.causal || key0 + KEYS - 1 <= sp.p0) &&
                             (a.window > 0 ? key0 > sp.p1 - a.window || key0 + KEYS <= a.sinks : key0 >= q.lo);
            float mx[2] = {m[0], m[1]};
#pragma unroll
            for (int nb = 0; nb < NB; ++nb)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    float x = sc[nb][j] * factor[j >> 1];
                    if (!all && !sees(a, q, pos[j >> 1], key0 + nb * 8 + (lane & 3) * 2 + (j & 1)))
                        x = -INFINITY;
                    sc[nb][j] = x;
                    mx[j >> 1] = fmaxf(mx[j >> 1], x);
                }
            float al[2];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                mx[h] = fmaxf(mx[h], __shfl_xor_sync(0xffffffffu, mx[h], 1));
                mx[h] = fmaxf(mx[h], __shfl_xor_sync(0xffffffffu, mx[h], 2));
                const float ms = mx[h] == -INFINITY ? 0.0f : mx[h];
                al[h] = ex2(m[h] - ms);
                m[h] = mx[h];
                mx[h] = ms - UP;
            }
            if (__any_sync(0xffffffffu, al[0] != 1.0f || al[1] != 1.0f)) {
#pragma unroll
                for (int d = 0; d < DP / 8; ++d) {
                    o[d][0] *= al[0]; o[d][1] *= al[0]; o[d][2] *= al[1]; o[d][3] *= al[1];
                }
                l[0] *= al[0];
                l[1] *= al[1];
            }
            uint32_t p[2 * NB];
#pragma unroll
            for (int nb = 0; nb < NB; ++nb)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const float e0 = ex2(sc[nb][2 * h] - mx[h]), e1 = ex2(sc[nb][2 * h + 1] - mx[h]);
                    l[h] += e0 + e1;
                    // weights in the cache's type (in 8 bits fp16) for the product: off by half a step,
                    // 2^-8 of a weight (bf16) or 2^-11, as the output's own rounding (fp16: at least
                    // 2^-25, 2^-39 of the largest weight); the sum keeps fp32
                    p[2 * nb + h] = pack2<M>(e0, e1);
                }
            if constexpr (QUANT) {
                code_product<DP, C>(ring_p + so + STAGE / 2, scales + SCALES / 2, per, p, o);
            } else {
#pragma unroll
                for (int d = 0; d < DP / 16; ++d) {
                    uint32_t b[4];
                    const int row = ml + (mi & 1) * 8, c = 2 * d + (mi >> 1);
                    ldm4t(b, vt + (c >> 3) * BLOCK + row * 128 + (((c & 7) ^ (row & 7)) * 16));
                    mma16816<T>(o[2 * d], p, b[0], b[1]);
                    mma16816<T>(o[2 * d + 1], p, b[2], b[3]);
                }
            }
            __syncwarp();                              // the stage may be overwritten
        }
        if (n > 0) done += n;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            l[h] += __shfl_xor_sync(0xffffffffu, l[h], 1);
            l[h] += __shfl_xor_sync(0xffffffffu, l[h], 2);
        }

        // ---- join the warps in the rings' memory
        __syncthreads();
        float* jm = reinterpret_cast<float*>(smem);    // [warp][16][MR], then [warp][16] maxima, sums
        float* jst = jm + RW_WARPS * RW_ROWS * MR;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int row = lane / 4 + 8 * h;
            float* dst = jm + (warp * RW_ROWS + row) * MR;
            if constexpr (QUANT) {
                code_row<DP>(o, h, dst);
            } else {
                dst += (lane & 3) * 2;
#pragma unroll
                for (int d = 0; d < DP / 8; ++d) {
                    dst[8 * d] = o[d][2 * h];
                    dst[8 * d + 1] = o[d][2 * h + 1];
                }
            }
            if ((lane & 3) == 0) {
                // fmaxf drops NaN, the sum keeps it: with an infinite maximum the row's share of
                // every join is NaN, so that a NaN score shows in the result
                jst[warp * RW_ROWS + row] = l[h] == l[h] ? m[h] - UP : INFINITY;
                jst[(RW_WARPS + warp) * RW_ROWS + row] = l[h];
            }
        }
        __syncthreads();
        auto stat = [&](int w, int row, int k) { return jst[(k * RW_WARPS + w) * RW_ROWS + row]; };
        auto value = [&](int w, int row, int c) {
            return *reinterpret_cast<const float4*>(jm + (w * RW_ROWS + row) * MR + 4 * c);
        };
        if (t0 == 0 && t1 == ld.tiles) {
            finish_rows<T, false>(a, q, kvh, row0, rows, RW_WARPS, stat, value, jst + 2 * RW_WARPS * RW_ROWS, &again);
            if (threadIdx.x == 0 && again) any_again = 1;
        } else {
            float* part = r.w.part + ((int64_t)blockIdx.x * 2 + (t0 == 0)) * RW_ROWS * (DP + 2);
            for (int i = threadIdx.x; i < rows * (DP / 4); i += RW_THREADS) {
                const int row = i / (DP / 4), c = i % (DP / 4);
                float mm = -INFINITY;
#pragma unroll
                for (int w = 0; w < RW_WARPS; ++w) mm = fmaxf(mm, stat(w, row, 0));
                const float ms = mm == -INFINITY ? 0.0f : mm;
                float4 x = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                float sum = 0.0f;
#pragma unroll
                for (int w = 0; w < RW_WARPS; ++w) {
                    const float wgt = ex2(stat(w, row, 0) - ms);
                    const float4 v = value(w, row, c);
                    x.x = fmaf(wgt, v.x, x.x); x.y = fmaf(wgt, v.y, x.y);
                    x.z = fmaf(wgt, v.z, x.z); x.w = fmaf(wgt, v.w, x.w);
                    sum = fmaf(wgt, stat(w, row, 1), sum);
                }
                *reinterpret_cast<float4*>(part + row * DP + 4 * c) = x;
                if (c == 0) {
                    part[RW_ROWS * DP + row] = mm;
                    part[RW_ROWS * (DP + 1) + row] = sum;
                }
            }
            if (t0 == 0 && threadIdx.x == 0) {
                r.w.joint[2 * blockIdx.x] = make_int4(s, kvh, rt, 1 + (int)((ld.tiles - t1 + share - 1) / share));
                r.w.joint[2 * blockIdx.x + 1] = make_int4(q.begin, q.n_new, q.kv, 0);
            }
        }
        cur += t1 - t0;
        fence_proxy_async_smem();                      // the next copies come behind these writes
        __syncthreads();
    }
    if (!any_again || abort) return;
    // ---- rows that came out not finite, of the units that are whole here (out of the way of the
    // loop: within it the decode batch took 349 us, not 345)
    pre = sh_pre;
    s = sh_seq;
    for (cur = blockIdx.x * share; cur < end;) {
        q = load_seq(a.b, a.max_kv, s, a.status);
        ld = seq_load<C>(r, q);
        if (cur >= pre + (int64_t)ld.units * ld.tiles) {
            pre += (int64_t)ld.units * ld.tiles;
            ++s;
            continue;
        }
        const int unit = (int)((cur - pre) / ld.tiles), t0 = (int)(cur - pre - (int64_t)unit * ld.tiles);
        const int n = (int)min((int64_t)(ld.tiles - t0), end - cur);
        if (n == ld.tiles) {                           // a warp's rows: four neighbours
            const int kvh = unit / ld.row_tiles, row0 = (unit - kvh * ld.row_tiles) * RW_ROWS;
            const int rows = (int)min((int64_t)RW_ROWS, (int64_t)q.n_new * a.group - row0);
            rows_exact<T, C>(a, q, kvh, row0, ((1u << rows) - 1u) & 0xfu << 4 * warp);
        }
        cur += n;
    }
}

// What both kernels left in pieces.  Blocks [0, rows_ctas): 16 rows each, of the unit begun
// in that CTA of the rows kernel; the rest: a group of 16 rows of a unit begun in a CTA of
// the chunk kernel.
struct JoinArgs {
    AttnArgs a;
    RowsWork rows;
    int rows_ctas, dp;
    ChunkJoin chunk;
};

template <typename T, int C>
__global__ void __launch_bounds__(RW_THREADS) paged_join_kernel(const __grid_constant__ JoinArgs j) {
    extern __shared__ float share[];
    __shared__ int again;
    asm volatile("griddepcontrol.wait;" ::: "memory");   // launched while the kernel before still runs
    const bool few = (int)blockIdx.x < j.rows_ctas;
    const int at = few ? blockIdx.x : blockIdx.x - j.rows_ctas;
    const int64_t c = few ? at : at / j.chunk.groups;
    const int r0 = few ? 0 : 16 * (at - (int)c * j.chunk.groups);
    const int4* joint = (few ? j.rows.joint : j.chunk.joint) + 2 * c;
    const int4 u = joint[0], x = joint[1];
    if (u.w == 0) return;
    const Seq q = j.a.b.shared ? shared_part(j.a.b, u.x) : seq_of(u.x, x.x, x.y, x.z);
    const int rows = few ? RW_ROWS : j.chunk.rows, row0 = u.z * rows + r0;
    const int64_t left = (int64_t)q.n_new * j.a.group - row0;
    if (left <= 0) return;
    const int64_t size = (int64_t)rows * (j.dp + 2);
    const float* part = (few ? j.rows.part : j.chunk.part) + c * 2 * size;
    finish_rows<T, true>(j.a, q, u.y, row0, (int)min((int64_t)16, left), u.w,
                   [&](int i, int row, int k) {
                       return part[(2 * i + (i == 0)) * size + rows * (j.dp + k) + r0 + row];
                   },
                   [&](int i, int row, int col) {   // rows: [row][DP]; chunk: [DP / 4][row][4]
                       return *reinterpret_cast<const float4*>(
                           part + (2 * i + (i == 0)) * size +
                           (few ? row * j.dp + 4 * col : (col * rows + r0 + row) * 4));
                   },
                   share, &again);
    if (again)   // (four neighbours a warp)
        attn_rows_exact<T, C, 1>(j.a, q, u.y, row0, (unsigned)again & 0xfu << 4 * (threadIdx.x >> 5));
}

inline int rows_dp(int64_t D) { return D <= 64 ? 64 : D <= 128 ? 128 : 256; }

template <int C>
int64_t rows_ctas(int dp, bool shared) {
    return (int64_t)device_sm_count() * (dp == 64    ? rows_ctas_per_sm<64, C>(shared)
                                         : dp == 128 ? rows_ctas_per_sm<128, C>(shared)
                                                     : rows_ctas_per_sm<256, C>(shared));
}

template <int C>
size_t rows_workspace(int dp, bool shared) {
    const size_t g = (size_t)rows_ctas<C>(dp, shared);
    return 2 * g * sizeof(int4) + g * 2 * RW_ROWS * (dp + 2) * sizeof(float);
}

template <typename T, int DP, int C, int CTAS>
hmm_status_t launch_rows(const RowsArgs& r, const CUtensorMap& k, const CUtensorMap& v, cudaStream_t st) {
    static std::atomic<uint64_t> done{0};
    constexpr size_t smem = rows_smem<DP, C, CTAS>();
    const hmm_status_t s = allow_smem(paged_rows_kernel<T, DP, C, CTAS>, smem, &done);
    if (s != HMM_OK) return s;
    return launch(paged_rows_kernel<T, DP, C, CTAS>, dim3((unsigned)(device_sm_count() * CTAS)), RW_THREADS, smem,
                  r.a.b.shared != nullptr, st, "paged_rows_kernel", k, v, r);
}

template <typename T, int C>
hmm_status_t run_rows(const RowsArgs& r, cudaStream_t st) {
    CUtensorMap k, v;
    hmm_status_t s = make_page_map(&k, r.a, r.a.k, r.box_rows, C != CODEC_NONE);
    if (s != HMM_OK) return s;
    s = make_page_map(&v, r.a, r.a.v, r.box_rows, C != CODEC_NONE);
    if (s != HMM_OK) return s;
    const int dp = rows_dp(r.a.D);
    if (dp == 64) return launch_rows<T, 64, C, 4>(r, k, v, st);
    if (dp == 256) return launch_rows<T, 256, C, 1>(r, k, v, st);
    if constexpr (C == CODEC_NONE) {
        if (!r.a.b.shared) return launch_rows<T, 128, C, 2>(r, k, v, st);
    }
    return launch_rows<T, 128, C, 3>(r, k, v, st);
}

template <typename T, int C>
hmm_status_t run_kernels(const AttnArgs& a, int max_new, unsigned char* ws, cudaStream_t st) {
    // A unit of up to 16 rows (one MMA's) reads its keys once either way and the many small
    // CTAs of the rows kernel keep more reads in flight; more rows would read them again
    // there: 64 rows of 4 KV heads over 5,000, 16 sequences, D = 128, 114 us there and 70 in
    // the chunk kernel, 32 rows 71 and 68 (over 777: 37 and 31, 31 in both).  In 8 bits, where the
    // chunk kernel has its codes widened beside the products, up to 32: 28 rows of 4 KV heads over
    // 700, 16 sequences, D = 128, 31 us there and 39 in the chunk kernel, over 5,000 49 and 52, 32
    // sequences over 16,000 154 and 203; 35 rows 33 and 39, 62 and 52, 211 and 203.  (A scale of zero
    // is the rows kernel's, which scales before it masks: in the chunk kernel a masked score of -inf
    // times zero would be NaN.)
    const bool chunk = chunk_applies(a) && a.scale_log2 != 0.0f;
    const int bound = a.b.shared ? a.b.n_tokens : max_new;       // (a group's rows are those of its sequences)
    const bool few = bound > 0 && (int64_t)std::min(bound, a.b.n_tokens) * a.group <= RW_ROWS;
    const bool with_rows = few || !chunk || (a.b.n_seq > 1 && a.min_rows <= rows_most<C>());
    const int most = !chunk || few ? INT32_MAX : rows_most<C>();      // rows of a sequence for the rows kernel
    const int dp = rows_dp(a.D);
    const int64_t ctas = rows_ctas<C>(dp, a.b.shared != nullptr);
    JoinArgs j{a, {(int4*)ws, (float*)(ws + 2 * (size_t)ctas * sizeof(int4))}, 0, dp, {}};
    hmm_status_t s;
    if (with_rows) {
        j.rows_ctas = (int)ctas;
        s = run_rows<T, C>(RowsArgs{a, j.rows, most, box_rows_of(a.page_tokens, rows_keys<C>()), wait_limit_ns()}, st);
        if (s != HMM_OK) return s;
    }
    if (chunk && !few) {
        s = run_chunk<C>(a, std::is_same<T, __nv_bfloat16>::value, with_rows ? most + 1 : 1, with_rows,
                      ws + up256(rows_workspace<C>(dp, a.b.shared != nullptr)), st, &j.chunk);
        if (s != HMM_OK) return s;
    }
    const int64_t blocks = j.rows_ctas + (int64_t)j.chunk.ctas * j.chunk.groups;
    if (blocks == 0) return HMM_OK;
    const size_t share = sizeof(float) * 32 * (std::max(j.rows_ctas, j.chunk.ctas) + 1);
    static std::atomic<uint64_t> done{0};
    s = allow_smem(paged_join_kernel<T, C>, sizeof(float) * 32 * 1024, &done);
    if (s != HMM_OK) return s;
    return launch(paged_join_kernel<T, C>, dim3((unsigned)blocks), RW_THREADS, share, true, st, "paged_join_kernel", j);
}

}  // namespace serve
}  // namespace hmm
