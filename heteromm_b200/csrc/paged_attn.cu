// paged_attn.cu — attention of ragged chunks of new tokens over a paged cache:
// the entry point, and the kernel for few rows (decoding, drafted tokens).
//
// paged_rows_kernel.  A unit is (sequence, KV head, 16 rows): rows are (new
// token, query head of the group), so grouped heads read their keys once.  With
// few rows the cache has to be read for next to no arithmetic and HBM bounds it;
// the design keeps reads in flight:
//   - all units' key tiles form one list, cut into as many equal pieces as CTAs
//     fit the GPU (ragged lengths balance by themselves); a CTA finds its piece
//     from the lengths on the device, so no host value goes stale;
//   - each warp owns 16 keys of a tile and its own ring of TMA stages, with no
//     barrier between warps: a box per 64 values of a page's rows (issued by as
//     many lanes as there are boxes, their page looked up one stage ahead), zeros
//     for the boxes that no row of the tile sees.  The copies cost a warp about 30
//     instructions a tile; with 16-byte cp.async (about 400) the issue slots bound
//     the kernel, not HBM;
//   - scores and the product with V on mma.sync (m16n8k16, fp32 sums), the
//     running maximum and sum in fp32 per warp, warps joined once per piece;
//   - a unit that several CTAs share leaves (maximum, sum, unnormalised rows) per
//     piece in the workspace, and paged_join_kernel adds the pieces in order.
// Measured: 64 sequences of up to 16,384 tokens, one new token each, 32 query and 8 KV
// heads of 128: 347-351 us, 6.3 TB/s (cp.async: 478); one token over 777: 11.9 us, of
// which 2.5 the join, over 4,000 17.6 us.
#include <algorithm>

#include "paged_attn.cuh"
#include "paged_attn_tc.cuh"

namespace hmm {
namespace serve {
using namespace sm100;
namespace {

constexpr int RW_WARPS = 4;
constexpr int RW_THREADS = 32 * RW_WARPS;
constexpr int RW_KEYS = 16;                   // keys of a warp's tile
constexpr int RW_TILE = RW_WARPS * RW_KEYS;   // keys of a CTA's tile
constexpr int RW_ROWS = 16;
constexpr int RW_STAGES = 3;

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

template <int DP>
constexpr int rows_ctas_per_sm() { return DP == 64 ? 4 : DP == 128 ? 2 : 1; }

template <int DP>
constexpr size_t rows_smem() {
    return 1024 + (size_t)RW_WARPS * RW_STAGES * 2 * RW_KEYS * DP * 2;
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

__device__ __forceinline__ Load seq_load(const RowsArgs& r, const Seq& q) {
    const int64_t rows = (int64_t)q.n_new * r.a.group;
    Load x{0, 0, 0};
    if (rows == 0 || rows > r.max_rows) return x;
    x.row_tiles = (int)((rows + RW_ROWS - 1) / RW_ROWS);
    x.units = x.row_tiles * r.a.hk;
    int64_t t = ((int64_t)q.kv + RW_TILE - 1) / RW_TILE;
    if (r.a.window > 0) {
        const int64_t near = ((int64_t)r.a.window + RW_ROWS + RW_TILE - 1) / RW_TILE + 1;
        t = min(t, near + ((int64_t)r.a.sinks + RW_TILE - 1) / RW_TILE);
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
template <typename T>
__device__ __noinline__ void rows_exact(const AttnArgs& a, int s, const Seq& q, int kvh, int row0, unsigned rows) {
    attn_rows_exact<T, 1>(a, s, q, kvh, row0, rows);
}

template <typename T, int DP>
__global__ void __launch_bounds__(RW_THREADS, rows_ctas_per_sm<DP>())
paged_rows_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV,
                  const __grid_constant__ RowsArgs r) {
    extern __shared__ __align__(1024) unsigned char smem_raw[];
    unsigned char* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
    __shared__ uint64_t full[RW_WARPS][RW_STAGES];
    __shared__ int64_t wt[RW_WARPS];
    __shared__ int64_t sh_pre;
    __shared__ int sh_seq, again, any_again, abort;
    constexpr int HALVES = DP / 64;                    // boxes of 64 values in a row
    constexpr int BLOCK = RW_KEYS * 128;               // 16 rows of 64 values, swizzled
    constexpr int STAGE = 2 * HALVES * BLOCK;          // K then V
    constexpr int MR = DP + 4;                         // joining rows: 4 banks apart
    // log2 of what weights are held by: the largest is 2^14 in fp16, whose range ends at 2^-25
    // (a key 18 nats below the largest had no weight at all, and a long tail of them a share
    // of the result).  It cancels against the sum, and lse takes it back with the maximum.
    constexpr float UP = std::is_same<T, __half>::value ? 14.0f : 0.0f;
    const AttnArgs& a = r.a;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
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
        const Load x = seq_load(r, q);
        own += (int64_t)x.units * x.tiles;
    });
    scan_incl(own, wt, &total);
    const int64_t per = max((int64_t)1, (total + gridDim.x - 1) / gridDim.x);
    int64_t cur = blockIdx.x * per;
    const int64_t end = min(total, cur + per);
    if (threadIdx.x == 0) r.w.joint[2 * blockIdx.x] = make_int4(0, 0, 0, 0);
    if (cur >= end) return;
    {
        int64_t run = 0;
        for (int s0 = 0; s0 < a.b.n_seq; s0 += RW_THREADS) {
            const int s = s0 + threadIdx.x;
            int64_t v = 0, sum;
            if (s < a.b.n_seq) {
                const Load x = seq_load(r, load_seq(a.b, a.max_kv, s, a.status));
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
    Load ld = seq_load(r, q);

    unsigned char* ring_p = smem + warp * RW_STAGES * STAGE;
    const uint32_t ring = smem_u32(ring_p);
    // lane: box rows [sub * box_rows, +box_rows) of the warp's 16 keys, and of the (K / V,
    // 64 values) boxes there every (32 / subs)-th
    const int subs = RW_KEYS / r.box_rows, sub = lane % subs, box0 = lane / subs, box_step = 32 / subs;
    uint32_t done = 0;                                 // tiles that the ring has seen
    bool dead = false;                                 // a wait gave up: no more copies
    while (cur < end) {
        while (cur >= pre + (int64_t)ld.units * ld.tiles) {
            pre += (int64_t)ld.units * ld.tiles;
            q = load_seq(a.b, a.max_kv, ++s, a.status);
            ld = seq_load(r, q);
        }
        const int unit = (int)((cur - pre) / ld.tiles);
        const int t0 = (int)(cur - pre - (int64_t)unit * ld.tiles);
        const int t1 = (int)min((int64_t)ld.tiles, t0 + (end - cur));
        const int kvh = unit / ld.row_tiles, rt = unit - kvh * ld.row_tiles;
        const int row0 = rt * RW_ROWS;
        const int rows = (int)min((int64_t)RW_ROWS, (int64_t)q.n_new * a.group - row0);
        const Span sp = tile_span(a, q, row0, row0 + rows);
        const int sink_tiles = (sp.sink + RW_TILE - 1) / RW_TILE;
        const int first = max(sp.lo / RW_TILE, sink_tiles);
        const int n_tiles = sink_tiles + max(0, (sp.hi + RW_TILE - 1) / RW_TILE - first);
        const int n = min(t1, n_tiles) - t0;           // tiles of this piece, <= 0: none

        auto key0_of = [&](int i) {                    // first key of this warp's part of tile t0 + i
            const int t = t0 + i;
            return (t < sink_tiles ? t : first + t - sink_tiles) * RW_TILE + warp * RW_KEYS;
        };
        int page = a.n_pages, row = 0;                 // this lane's box rows of the next tile
        auto lookup = [&](int i) {
            page = a.n_pages;                          // out of range: zeros
            if (i < n) {
                const int k0 = key0_of(i) + sub * r.box_rows;
                if (k0 < sp.sink || (k0 + r.box_rows > sp.lo && k0 < sp.hi)) {
                    const int lp = a.by_page(k0);
                    const int e = page_of(a, s, lp);
                    if (e >= 0) {
                        page = e;
                        row = k0 - lp * a.page_tokens;
                    }
                }
            }
        };
        auto issue = [&](int i) {                      // copies of tile i, whose lookup is in page / row
            if (i < n && !dead) {
                const uint32_t st = (done + i) % RW_STAGES;
                if (lane == 0) mbar_expect_tx(&full[warp][st], STAGE);
                __syncwarp();
                const uint32_t d = ring + st * STAGE + sub * r.box_rows * 128;
#pragma unroll 2
                for (int b = box0; b < 2 * HALVES; b += box_step)
                    tma_load_page(d + b * BLOCK, b < HALVES ? &tmK : &tmV, &full[warp][st],
                                  64 * (b < HALVES ? b : b - HALVES), row, kvh, page);
            }
        };

        // q fragments: rows lane / 4 and lane / 4 + 8
        uint32_t qf[DP / 16][4];
        int pos[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int row = lane / 4 + 8 * h;
            const bool real = row < rows;
            const int at = row0 + (real ? row : 0);
            pos[h] = real ? row_pos(a, q, at) : -1;
            const unsigned char* src = a.q + (int64_t)(q.begin + at / a.group) * a.q_token +
                                       (int64_t)(kvh * a.group + at % a.group) * a.q_head;
#pragma unroll
            for (int k = 0; k < DP / 16; ++k)
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    const int d = k * 16 + j * 8 + (lane & 3) * 2;
                    qf[k][h + 2 * j] = real && d < a.D ? __ldg(reinterpret_cast<const uint32_t*>(src + 2 * d)) : 0u;
                }
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
            const uint32_t kt = ring + so, vt = kt + HALVES * BLOCK;
            const int key0 = key0_of(i);
            if (!(key0 >= sp.lo && key0 + RW_KEYS <= sp.hi) && key0 + RW_KEYS > sp.sink) {
                // V rows that no row of the unit sees, beside some that are seen, become
                // zeros: a weight of zero times what a slot of nobody holds is only zero then
                if (lane < RW_KEYS && !span_has(sp, key0 + lane)) {
#pragma unroll
                    for (int c = 0; c < HALVES * 8; ++c)
                        *reinterpret_cast<uint4*>(ring_p + so + (HALVES + (c >> 3)) * BLOCK + lane * 128 + (c & 7) * 16) =
                            make_uint4(0u, 0u, 0u, 0u);
                }
                __syncwarp();
            }
            float sc[2][4] = {};
            const int mi = lane >> 3, ml = lane & 7;
#pragma unroll
            for (int k = 0; k < DP / 16; ++k) {
                uint32_t b[4];
                const int row = ml + (mi >> 1) * 8, c = 2 * k + (mi & 1);
                ldm4(b, kt + (c >> 3) * BLOCK + row * 128 + (((c & 7) ^ (row & 7)) * 16));
                mma16816<T>(sc[0], qf[k], b[0], b[1]);
                mma16816<T>(sc[1], qf[k], b[2], b[3]);
            }
            const bool all = key0 + RW_KEYS <= q.kv && (!a.causal || key0 + RW_KEYS - 1 <= sp.p0) &&
                             (a.window <= 0 || key0 > sp.p1 - a.window || key0 + RW_KEYS <= a.sinks);
            float mx[2] = {m[0], m[1]};
#pragma unroll
            for (int nb = 0; nb < 2; ++nb)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    float x = sc[nb][j] * a.scale_log2;
                    if (!all && !sees(a, q.kv, pos[j >> 1], key0 + nb * 8 + (lane & 3) * 2 + (j & 1)))
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
            uint32_t p[4];
#pragma unroll
            for (int nb = 0; nb < 2; ++nb)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const float e0 = ex2(sc[nb][2 * h] - mx[h]), e1 = ex2(sc[nb][2 * h + 1] - mx[h]);
                    l[h] += e0 + e1;
                    // weights in the cache's type for the product: off by half a step, 2^-8 of a
                    // weight (bf16) or 2^-11, as the output's own rounding; the sum keeps fp32
                    p[2 * nb + h] = pack2<T>(e0, e1);
                }
#pragma unroll
            for (int d = 0; d < DP / 16; ++d) {
                uint32_t b[4];
                const int row = ml + (mi & 1) * 8, c = 2 * d + (mi >> 1);
                ldm4t(b, vt + (c >> 3) * BLOCK + row * 128 + (((c & 7) ^ (row & 7)) * 16));
                mma16816<T>(o[2 * d], p, b[0], b[1]);
                mma16816<T>(o[2 * d + 1], p, b[2], b[3]);
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
            float* dst = jm + (warp * RW_ROWS + row) * MR + (lane & 3) * 2;
#pragma unroll
            for (int d = 0; d < DP / 8; ++d) {
                dst[8 * d] = o[d][2 * h];
                dst[8 * d + 1] = o[d][2 * h + 1];
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
            finish_rows<T, false>(a, s, q, kvh, row0, rows, RW_WARPS, stat, value, jst + 2 * RW_WARPS * RW_ROWS, &again);
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
                r.w.joint[2 * blockIdx.x] = make_int4(s, kvh, rt, 1 + (int)((ld.tiles - t1 + per - 1) / per));
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
    for (cur = blockIdx.x * per; cur < end;) {
        q = load_seq(a.b, a.max_kv, s, a.status);
        ld = seq_load(r, q);
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
            rows_exact<T>(a, s, q, kvh, row0, ((1u << rows) - 1u) & 0xfu << 4 * warp);
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

template <typename T>
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
    const Seq q{x.x, x.y, x.z, true};
    const int rows = few ? RW_ROWS : j.chunk.rows, row0 = u.z * rows + r0;
    const int64_t left = (int64_t)q.n_new * j.a.group - row0;
    if (left <= 0) return;
    const int64_t size = (int64_t)rows * (j.dp + 2);
    const float* part = (few ? j.rows.part : j.chunk.part) + c * 2 * size;
    finish_rows<T, true>(j.a, u.x, q, u.y, row0, (int)min((int64_t)16, left), u.w,
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
        attn_rows_exact<T, 1>(j.a, u.x, q, u.y, row0, (unsigned)again & 0xfu << 4 * (threadIdx.x >> 5));
}

int rows_dp(int64_t D) { return D <= 64 ? 64 : D <= 128 ? 128 : 256; }

int64_t rows_ctas(int dp) {
    return (int64_t)device_sm_count() * (dp == 64 ? rows_ctas_per_sm<64>() : dp == 128 ? rows_ctas_per_sm<128>() : 1);
}

size_t up256(size_t v) { return (v + 255) & ~size_t(255); }

size_t rows_workspace(int dp) {
    const size_t g = (size_t)rows_ctas(dp);
    return 2 * g * sizeof(int4) + g * 2 * RW_ROWS * (dp + 2) * sizeof(float);
}

template <typename T, int DP>
hmm_status_t launch_rows(const RowsArgs& r, const CUtensorMap& k, const CUtensorMap& v, cudaStream_t st) {
    static std::atomic<uint64_t> done{0};
    const hmm_status_t s = allow_smem(paged_rows_kernel<T, DP>, rows_smem<DP>(), &done);
    if (s != HMM_OK) return s;
    return launch(paged_rows_kernel<T, DP>, dim3((unsigned)rows_ctas(DP)), RW_THREADS, rows_smem<DP>(), false, st,
                  "paged_rows_kernel", k, v, r);
}

template <typename T>
hmm_status_t run_rows(const RowsArgs& r, cudaStream_t st) {
    CUtensorMap k, v;
    hmm_status_t s = make_page_map(&k, r.a, r.a.k, r.box_rows);
    if (s != HMM_OK) return s;
    s = make_page_map(&v, r.a, r.a.v, r.box_rows);
    if (s != HMM_OK) return s;
    const int dp = rows_dp(r.a.D);
    return dp == 64 ? launch_rows<T, 64>(r, k, v, st) : dp == 128 ? launch_rows<T, 128>(r, k, v, st)
                                                                  : launch_rows<T, 256>(r, k, v, st);
}

template <typename T>
hmm_status_t run_attention(const AttnArgs& a, int max_new, unsigned char* ws, cudaStream_t st) {
    // A unit of up to 16 rows (one MMA's) reads its keys once either way and the many small
    // CTAs of the rows kernel keep more reads in flight; more rows would read them again
    // there: 64 rows of 4 KV heads over 5,000, 16 sequences, D = 128, 113 us there and 69 in
    // the chunk kernel, 32 rows 67 in both (over 777: 34 and 30, 25 and 29).  (A scale of zero is the rows kernel's, which scales before it masks: in the
    // chunk kernel a masked score of -inf times zero would be NaN.)
    const bool chunk = chunk_applies(a) && a.scale_log2 != 0.0f;
    const bool few = max_new > 0 && (int64_t)std::min(max_new, a.b.n_tokens) * a.group <= RW_ROWS;
    const bool with_rows = few || !chunk || a.b.n_seq > 1;
    const int most = !chunk || few ? INT32_MAX : RW_ROWS;      // rows of a sequence for the rows kernel
    const int dp = rows_dp(a.D);
    const int64_t ctas = rows_ctas(dp);
    JoinArgs j{a, {(int4*)ws, (float*)(ws + 2 * (size_t)ctas * sizeof(int4))}, 0, dp, {}};
    hmm_status_t s;
    if (with_rows) {
        j.rows_ctas = (int)ctas;
        s = run_rows<T>(RowsArgs{a, j.rows, most, box_rows_of(a.page_tokens, RW_KEYS), wait_limit_ns()}, st);
        if (s != HMM_OK) return s;
    }
    if (chunk && !few) {
        s = run_chunk(a, std::is_same<T, __nv_bfloat16>::value, with_rows ? most + 1 : 1, with_rows,
                      ws + up256(rows_workspace(dp)), st, &j.chunk);
        if (s != HMM_OK) return s;
    }
    const int64_t blocks = j.rows_ctas + (int64_t)j.chunk.ctas * j.chunk.groups;
    if (blocks == 0) return HMM_OK;
    const size_t share = sizeof(float) * 32 * (std::max(j.rows_ctas, j.chunk.ctas) + 1);
    static std::atomic<uint64_t> done{0};
    s = allow_smem(paged_join_kernel<T>, sizeof(float) * 32 * 1024, &done);
    if (s != HMM_OK) return s;
    return launch(paged_join_kernel<T>, dim3((unsigned)blocks), RW_THREADS, share, true, st, "paged_join_kernel", j);
}

}  // namespace
}  // namespace serve
}  // namespace hmm

using namespace hmm;
using namespace hmm::serve;

extern "C" size_t hmm_paged_attention_workspace_size(int64_t n_seq, int64_t n_tokens, int64_t n_heads,
                                                     int64_t n_kv_heads, int64_t D) {
    if (n_seq < 0 || n_tokens < 0 || n_heads < 1 || n_kv_heads < 1 || D < 1 || D > 256) return 0;
    const int dp = rows_dp(D);
    return up256(rows_workspace(dp)) + chunk_workspace(n_seq, n_tokens, n_heads, n_kv_heads, D);
}

extern "C" hmm_status_t hmm_paged_attention(const hmm_paged_cache_t* cache, const hmm_paged_batch_t* batch,
                                            const void* q, int64_t q_token, int64_t q_head,
                                            int64_t n_heads, float scale, int causal, int64_t window,
                                            int64_t sinks, int64_t max_new, void* out, float* lse,
                                            int32_t* device_status, void* workspace,
                                            size_t workspace_bytes, void* stream) {
    AttnArgs a{};
    hmm_status_t s = check_batch(cache, batch, &a.b, &a.k, &a.v);
    if (s != HMM_OK) return s;
    HMM_REQUIRE(cache->D <= 256, "D must be a multiple of 8 in [8, 256], got %lld", (long long)cache->D);
    HMM_REQUIRE(n_heads >= 1 && n_heads <= 65535 && n_heads % cache->n_kv_heads == 0,
                "n_heads must be a multiple of n_kv_heads in [1, 65535], got %lld", (long long)n_heads);
    HMM_REQUIRE(device_status, "null device_status");
    HMM_REQUIRE(window >= 0 && sinks >= 0, "window and sinks must be >= 0");
    HMM_REQUIRE(causal || (window == 0 && sinks == 0), "a window and sinks need causal attention");
    HMM_REQUIRE(max_new >= 0, "max_new must be >= 0");
    HMM_REQUIRE(q_token >= 0 && q_token % 8 == 0 && q_head >= 0 && q_head % 8 == 0,
                "q strides must be multiples of 8 elements");
    HMM_REQUIRE(batch->n_tokens * n_heads / cache->n_kv_heads < (int64_t(1) << 31),
                "n_tokens * (n_heads / n_kv_heads) must be < 2^31");
    if (batch->n_seq == 0 || batch->n_tokens == 0) return HMM_OK;
    HMM_REQUIRE(cache->n_pages >= 1, "the cache has no pages");
    HMM_REQUIRE(batch->pages_per_seq * cache->page_tokens <= (int64_t(1) << 31) - 1024,
                "pages_per_seq * page_tokens must be <= 2^31 - 1024");   // ends of tiles stay in 31 bits
    const int64_t steps[6] = {cache->page_tokens > 1 ? cache->k_token : 8, cache->n_kv_heads > 1 ? cache->k_head : 8,
                              cache->n_pages > 1 ? cache->k_page : 8, cache->page_tokens > 1 ? cache->v_token : 8,
                              cache->n_kv_heads > 1 ? cache->v_head : 8, cache->n_pages > 1 ? cache->v_page : 8};
    for (int64_t x : steps)
        HMM_REQUIRE(x > 0 && x < (int64_t(1) << 39), "cache strides must be in [8, 2^39) elements, got %lld",
                    (long long)x);
    HMM_REQUIRE(q && out, "null q or out");
    HMM_REQUIRE(aligned16(q) && aligned16(out), "q and out must be 16-byte aligned");
    const size_t need = hmm_paged_attention_workspace_size(batch->n_seq, batch->n_tokens, n_heads,
                                                           cache->n_kv_heads, cache->D);
    if (!workspace || workspace_bytes < need)
        return set_error(HMM_ERR_OOM, "workspace too small: %zu < %zu", workspace_bytes, need);
    HMM_REQUIRE(aligned16(workspace), "workspace must be 16-byte aligned");
    const uintptr_t q0 = (uintptr_t)q, o0 = (uintptr_t)out;
    HMM_REQUIRE(o0 >= q0 + 2 * (size_t)((batch->n_tokens - 1) * q_token + (n_heads - 1) * q_head + cache->D) ||
                    q0 >= o0 + 2 * (size_t)(batch->n_tokens * n_heads * cache->D),
                "out overlaps q");   // rows are read again where they come out not finite
    a.q = (const unsigned char*)q;
    a.q_token = 2 * q_token;
    a.q_head = 2 * q_head;
    a.out = (unsigned char*)out;
    a.lse = lse;
    a.scale = scale;
    a.scale_log2 = scale * 1.44269504088896340736f;
    a.causal = causal != 0;
    a.max_kv = batch->pages_per_seq * cache->page_tokens;
    a.window = window < a.max_kv ? (int)window : 0;   // a window over everything is none
    a.sinks = (int)std::min<int64_t>(sinks, a.max_kv);
    a.hq = (int)n_heads;
    a.hk = (int)cache->n_kv_heads;
    a.group = a.hq / a.hk;
    a.by_group = FastDiv::of(a.group);
    a.by_page = FastDiv::of((int)cache->page_tokens);
    a.D = (int)cache->D;
    a.page_tokens = (int)cache->page_tokens;
    a.n_pages = (int)cache->n_pages;
    a.status = device_status;
    const int hint = (int)std::min<int64_t>(max_new, INT32_MAX);
    return cache->dtype == HMM_DTYPE_BF16
               ? run_attention<__nv_bfloat16>(a, hint, (unsigned char*)workspace, (cudaStream_t)stream)
               : run_attention<__half>(a, hint, (unsigned char*)workspace, (cudaStream_t)stream);
}
