// paged_append.cuh — the kernel of the step before attention over a paged cache: RMS norm
// of every query and key head, position rotation, and the store of keys and values into
// the cache's pages, as 16-bit values or in 8 bits.
//
//   y = x / sqrt(mean(x^2) + eps) * w        (without a weight y = x)
//   (a, b) -> (a cos - b sin, b cos + a sin) on pairs of the first rotary_dim
//   values: neighbours (2i, 2i+1), or halves (i, i + rotary_dim / 2)
//
// The pass has to read and write every value once (2 B each way) and does a
// handful of fp32 operations on it: HBM and, at 16 values a lane and ~300
// instructions a step, the issue slots bound it.  A warp keeps a list of tokens
// and goes through each one's rows in steps (as many rows of one kind as its lane
// groups hold); the loads of the next steps, over the token's end too, are in
// flight meanwhile, and the token's sequence, page and angles are looked up once.
// Few tokens are shared by several warps, down to a step each.  Two steps in
// flight at 5 blocks per SM measured best (8,198 tokens of 48 heads of 128: 53 us,
// 3.9 TB/s; 4 at 4 blocks 60 us; a block per token, without lists, 66 us).
// A head's row lies in a group of 2^n lanes with one or two 16-byte vectors
// each; the sum of squares is a butterfly in the group.  The partner of a halves
// pair is in the lane's other vector (a head turned as a whole), a shuffle away
// (rotary_dim a multiple of 16), or goes through shared memory.  A lane's angles
// are the same for every head.  Everything is computed in fp32 and rounded once.
// A cache in 8 bits (C): a group of 32 values is four neighbouring lanes' vectors, its
// largest magnitude two shuffles, and a lane stores 8 bytes of codes (8,198 tokens of 48 heads of
// 128, fp16 to int8, neighbouring pairs: 70 us at 4 blocks per SM, 75 at 5, 90 at 3).
#pragma once

#include <type_traits>

#include "paged_quant.cuh"

namespace hmm {
namespace serve {

constexpr int AP_THREADS = 128;
// Blocks per SM; codes take more registers.
constexpr int ap_minb(bool quant) { return quant ? 4 : 5; }
constexpr int AP_DEPTH = 2;      // steps whose loads are in flight

enum RopeMode { ROPE_NONE, ROPE_PAIRS, ROPE_HALVES, ROPE_HALVES_LANE, ROPE_HALVES_SMEM };

struct Rows {                    // one of q, k, v, q_out: strides in bytes
    unsigned char* base;
    int64_t token, head;
};

struct AppendArgs {
    Batch b;
    Pages k_pages, v_pages;
    Rows q, k, v, out;
    const void* w[2];            // norm weights of q and k, or null
    bool w_f32;
    const float* rope;           // [n_pos][half][2]
    const int32_t* positions;    // [n_tokens] or null
    int64_t n_pos;
    int64_t max_kv;
    int n_pages;
    int hq, hk, D, vecs, half, page_tokens;
    QuantRows quant;             // (C != CODEC_NONE)
    int lpr_log2;                // lanes of a row's group
    int steps_q, steps_k;        // a token's steps of queries, and of keys or values
    int parts;                   // warps that share a token's steps
    int tokens_at_once;          // tokens that the grid's warps hold at once
    float eps, inv_d;
    int32_t* status;
};

// Pairs of fp32 values: one instruction for both.
__device__ __forceinline__ uint64_t f2(float lo, float hi) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
    return r;
}
__device__ __forceinline__ float2 un2(uint64_t v) {
    float2 r;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
    return r;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
    uint64_t d;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
    return d;
}

template <typename T>
__device__ __forceinline__ void unpack4(const uint4& w, uint64_t* f) {
    const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 p = unpack2<T>(u[i]);
        f[i] = f2(p.x, p.y);
    }
}

template <typename T>
__device__ __forceinline__ uint4 pack4(const uint64_t* f) {
    uint32_t u[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 p = un2(f[i]);
        u[i] = pack2<T>(p.x, p.y);
    }
    return make_uint4(u[0], u[1], u[2], u[3]);
}

// A warp's place in its list: token t, step `it` of the token's steps.  A step is
// the rows of one kind that a warp's lane groups hold at once.
struct Cursor {
    int t, it;
};

template <typename T, int VPL, int MODE, int C>
__global__ void __launch_bounds__(AP_THREADS, ap_minb(C != CODEC_NONE)) paged_append_kernel(const __grid_constant__ AppendArgs a) {
    extern __shared__ float sm[];   // ROPE_HALVES_SMEM: a row of D values per group
    const int lane = threadIdx.x & 31;
    const int id = blockIdx.x * (AP_THREADS / 32) + (threadIdx.x >> 5);
    const int part = id % a.parts;
    const int lpr = 1 << a.lpr_log2, n_groups = 32 >> a.lpr_log2, group = lane >> a.lpr_log2,
              gl = lane & (lpr - 1);
    const int steps = a.steps_q + 2 * a.steps_k;
    auto next = [&](Cursor& c) {
        if ((c.it += a.parts) >= steps) {
            c.it = part;
            c.t += a.tokens_at_once;
        }
    };
    auto kind_of = [&](int it) { return it < a.steps_q ? 0 : it < a.steps_q + a.steps_k ? 1 : 2; };
    auto head_of = [&](int it, int kind) {
        return (it - (kind == 0 ? 0 : kind == 1 ? a.steps_q : a.steps_q + a.steps_k)) * n_groups + group;
    };
    Cursor at{id / a.parts, part};
    if (at.t >= a.tokens_at_once) return;
    Cursor ahead = at;
    uint4 x[AP_DEPTH][VPL];
    auto load = [&](uint4* v) {     // the rows of `ahead`, which moves on
        if (ahead.t >= a.b.n_tokens) return;
        const int kind = kind_of(ahead.it), h = head_of(ahead.it, kind);
        const Rows& in = kind == 0 ? a.q : kind == 1 ? a.k : a.v;
        const unsigned char* src = in.base + ahead.t * in.token + h * in.head + 16 * gl;
#pragma unroll
        for (int j = 0; j < VPL; ++j)
            v[j] = h < (kind == 0 ? a.hq : a.hk) && gl + j * lpr < a.vecs
                       ? *reinterpret_cast<const uint4*>(src + 16 * j * lpr)
                       : make_uint4(0u, 0u, 0u, 0u);
        next(ahead);
    };
#pragma unroll
    for (int u = 0; u < AP_DEPTH; ++u) load(x[u]);

    int token = -1, weight_of = -1;
    bool ok = false;
    int slot = 0;
    int64_t phys = 0;
    const void* w = nullptr;
    uint64_t wf[VPL][4];
    // The angles of the lane's values, the same for every row.  ROPE_PAIRS: (cos, cos) and
    // (-sin, sin) of each pair.  Else of values 2 i, 2 i + 1 as pairs, for the first vector
    // alone where the second holds the partners.
    constexpr int CV = MODE == ROPE_HALVES_LANE ? 1 : VPL;
    uint64_t c[CV][4], sn[CV][4];

    // The place and angles of token t; false for a padding row and one that is flagged.
    auto place = [&](int t) {
        const int s = warp_find_seq(a.b, t);
        const int begin = __ldg(a.b.cu + s), end = __ldg(a.b.cu + s + 1), kv = __ldg(a.b.kv_len + s);
        if (t < begin || t >= end) {
            // a padding row, left as it is (or cu_new is not ascending)
            if (lane == 0 && t >= __ldg(a.b.cu) && t < __ldg(a.b.cu + a.b.n_seq))
                atomicOr(a.status, HMM_STATUS_BATCH_BOUNDS);
            return false;
        }
        const int64_t p = (int64_t)kv - (end - begin) + (t - begin);
        const int64_t ap = MODE == ROPE_NONE ? 0 : a.positions ? (int64_t)__ldg(a.positions + t) : p;
        if (begin < 0 || end > a.b.n_tokens || kv < 0 || kv > a.max_kv || p < 0 ||
            (MODE != ROPE_NONE && (ap < 0 || ap >= a.n_pos))) {
            if (lane == 0) atomicOr(a.status, HMM_STATUS_BATCH_BOUNDS);
            return false;
        }
        const int logical = (int)p / a.page_tokens;
        slot = (int)p - logical * a.page_tokens;
        phys = __ldg(a.b.table + (int64_t)s * a.b.pages_per_seq + logical);
        if (phys < 0 || phys >= a.n_pages) {
            if (lane == 0) atomicOr(a.status, HMM_STATUS_PAGE_BOUNDS);
            return false;
        }
        if (MODE != ROPE_NONE) {
            const float2* row = reinterpret_cast<const float2*>(a.rope) + ap * a.half;
#pragma unroll
            for (int j = 0; j < CV; ++j)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int e = 8 * (gl + j * lpr) + 2 * i;
                    if (MODE == ROPE_PAIRS) {   // a' = a c - b s, b' = b c + a s on (a, b)
                        const float2 cs = e < 2 * a.half ? __ldg(row + (e >> 1)) : make_float2(1.0f, 0.0f);
                        c[j][i] = f2(cs.x, cs.x);
                        sn[j][i] = f2(-cs.y, cs.y);
                    } else {                    // each value times cos, its partner times -sin (first half) or sin
                        float2 cs[2];
#pragma unroll
                        for (int k = 0; k < 2; ++k)
                            cs[k] = e + k < 2 * a.half ? __ldg(row + (e + k < a.half ? e + k : e + k - a.half))
                                                       : make_float2(1.0f, 0.0f);
                        c[j][i] = f2(cs[0].x, cs[1].x);
                        sn[j][i] = f2(e < a.half ? -cs[0].y : cs[0].y, e + 1 < a.half ? -cs[1].y : cs[1].y);
                    }
                }
        }
        return true;
    };

    auto step = [&](const uint4* v) {   // the rows of `at`
        if (at.t != token) {
            token = at.t;
            ok = place(token);
        }
        if (!ok) return;
        const int kind = kind_of(at.it), h = head_of(at.it, kind);
        const bool live = h < (kind == 0 ? a.hq : a.hk);
        const Pages& pg = kind == 1 ? a.k_pages : a.v_pages;
        unsigned char* dst = (kind == 0 ? a.out.base + token * a.out.token + h * a.out.head
                                        : pg.base + phys * pg.page + slot * pg.token + h * pg.head) + 16 * gl;
        if (C == CODEC_NONE && kind == 2) {   // values are stored as they are
#pragma unroll
            for (int j = 0; j < VPL; ++j)
                if (live && gl + j * lpr < a.vecs) *reinterpret_cast<uint4*>(dst + 16 * j * lpr) = v[j];
            return;
        }
        // Rows of a cache in 8 bits: all lanes of the warp, for the shuffles.
        auto store_codes = [&](const uint64_t (*y)[4]) {
            unsigned char* block = pg.base + phys * pg.page + h * pg.head;
#pragma unroll
            for (int j = 0; j < VPL; ++j) {
                const int vec = gl + j * lpr;
                float f[8];
                uint32_t top = 0;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float2 p = un2(y[j][i]);
                    f[2 * i] = p.x;
                    f[2 * i + 1] = p.y;
                    top = max(top, max(__float_as_uint(p.x) & 0x7fffffffu, __float_as_uint(p.y) & 0x7fffffffu));
                }
                top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
                top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
                const int s = scale_byte<C>(top);
                const float inv = __uint_as_float((uint32_t)(254 - s) << 23);   // 2^(127 - s)
#pragma unroll
                for (int i = 0; i < 8; ++i) f[i] = s == 255 ? 0.0f : f[i] * inv;
                if (!live || vec >= a.vecs) continue;
                *reinterpret_cast<uint2*>(block + slot * pg.token + 8 * vec) =
                    make_uint2(codes4<C>(f[0], f[1], f[2], f[3]), codes4<C>(f[4], f[5], f[6], f[7]));
                if ((vec & 3) == 0) block[a.quant.scales + (int64_t)slot * a.quant.per_token + (vec >> 2)] = (unsigned char)s;
            }
        };
        if (C != CODEC_NONE && kind == 2) {
            uint64_t y[VPL][4];
#pragma unroll
            for (int j = 0; j < VPL; ++j) unpack4<T>(v[j], y[j]);
            store_codes(y);
            return;
        }
        if (kind != weight_of) {
            weight_of = kind;
            w = a.w[kind];
#pragma unroll
            for (int j = 0; j < VPL; ++j) {
                const int vi = min(gl + j * lpr, a.vecs - 1);
                if (!w) {
                } else if (a.w_f32) {
                    const float4* p = reinterpret_cast<const float4*>(w) + 2 * vi;
                    const float4 lo = __ldg(p), hi = __ldg(p + 1);
                    wf[j][0] = f2(lo.x, lo.y); wf[j][1] = f2(lo.z, lo.w);
                    wf[j][2] = f2(hi.x, hi.y); wf[j][3] = f2(hi.z, hi.w);
                } else {
                    unpack4<T>(__ldg(reinterpret_cast<const uint4*>(w) + vi), wf[j]);
                }
            }
        }
        uint64_t y[VPL][4];
#pragma unroll
        for (int j = 0; j < VPL; ++j) unpack4<T>(v[j], y[j]);
        if (w) {
            uint64_t s2 = mul2(y[0][0], y[0][0]);
#pragma unroll
            for (int j = 0; j < VPL; ++j)
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (i + j > 0) s2 = fma2(y[j][i], y[j][i], s2);
            const float2 s1 = un2(s2);
            float ss = s1.x + s1.y;
            for (int o = lpr >> 1; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
            const float inv = rsqrtf(fmaf(ss, a.inv_d, a.eps));
            const uint64_t inv2 = f2(inv, inv);
#pragma unroll
            for (int j = 0; j < VPL; ++j)
#pragma unroll
                for (int i = 0; i < 4; ++i) y[j][i] = mul2(mul2(y[j][i], inv2), wf[j][i]);
        }
        if (MODE == ROPE_PAIRS) {
#pragma unroll
            for (int j = 0; j < VPL; ++j)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    if (8 * (gl + j * lpr) + 2 * i >= 2 * a.half) continue;   // as it is, infinities too
                    const float2 ab = un2(y[j][i]);
                    y[j][i] = fma2(f2(ab.y, ab.x), sn[j][i], mul2(y[j][i], c[j][i]));
                }
        } else if (MODE == ROPE_HALVES_LANE) {
            // vectors gl and gl + lpr of the row: value e and its partner e + half
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint64_t p0 = y[0][i], p1 = y[VPL - 1][i];
                const float2 sv = un2(sn[0][i]);
                y[0][i] = fma2(p1, sn[0][i], mul2(p0, c[0][i]));
                y[VPL - 1][i] = fma2(p0, f2(-sv.x, -sv.y), mul2(p1, c[0][i]));
            }
        } else if (MODE == ROPE_HALVES) {
            // vector gl holds values [8 gl, 8 gl + 8); half is a multiple of 8
            const int hv = a.half >> 3;
            const bool turned = gl < 2 * hv;
            const int partner = gl < hv ? gl + hv : turned ? gl - hv : gl;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float2 ab = un2(y[0][i]);
                const float o0 = __shfl_sync(0xffffffffu, ab.x, partner, lpr);
                const float o1 = __shfl_sync(0xffffffffu, ab.y, partner, lpr);
                if (turned) y[0][i] = fma2(f2(o0, o1), sn[0][i], mul2(y[0][i], c[0][i]));
            }
        } else if (MODE == ROPE_HALVES_SMEM) {
            float* row = sm + ((threadIdx.x >> 5) * n_groups + group) * a.D;
#pragma unroll
            for (int j = 0; j < VPL; ++j) {
                const int vi = gl + j * lpr;
                if (vi < a.vecs) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const float2 ab = un2(y[j][i]);
                        row[8 * vi + 2 * i] = ab.x;
                        row[8 * vi + 2 * i + 1] = ab.y;
                    }
                }
            }
            __syncwarp();
#pragma unroll
            for (int j = 0; j < VPL; ++j)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int e = 8 * (gl + j * lpr) + 2 * i;
                    const float2 ab = un2(y[j][i]), cc = un2(c[j][i]), ss = un2(sn[j][i]);
                    float2 r = ab;
                    if (e < 2 * a.half) r.x = ab.x * cc.x + row[e < a.half ? e + a.half : e - a.half] * ss.x;
                    if (e + 1 < 2 * a.half)
                        r.y = ab.y * cc.y + row[e + 1 < a.half ? e + 1 + a.half : e + 1 - a.half] * ss.y;
                    y[j][i] = f2(r.x, r.y);
                }
            __syncwarp();
        }
        if (C != CODEC_NONE && kind == 1) {
            store_codes(y);
        } else if (live) {
#pragma unroll
            for (int j = 0; j < VPL; ++j)
                if (gl + j * lpr < a.vecs) *reinterpret_cast<uint4*>(dst + 16 * j * lpr) = pack4<T>(y[j]);
        }
    };
    while (at.t < a.b.n_tokens) {
#pragma unroll
        for (int u = 0; u < AP_DEPTH; ++u) {
            if (at.t >= a.b.n_tokens) break;
            step(x[u]);
            load(x[u]);
            next(at);
        }
    }
}

template <typename T, int VPL, int C>
hmm_status_t launch_append(const AppendArgs& a, int mode, cudaStream_t st) {
    const int64_t warps = (int64_t)a.tokens_at_once * a.parts;
    const unsigned grid = (unsigned)((warps + AP_THREADS / 32 - 1) / (AP_THREADS / 32));
    const size_t smem = mode == ROPE_HALVES_SMEM ? sizeof(float) * (AP_THREADS >> a.lpr_log2) * a.D : 0;
    constexpr int threads = AP_THREADS;
    switch (mode) {
        case ROPE_NONE: paged_append_kernel<T, VPL, ROPE_NONE, C><<<grid, threads, 0, st>>>(a); break;
        case ROPE_PAIRS: paged_append_kernel<T, VPL, ROPE_PAIRS, C><<<grid, threads, 0, st>>>(a); break;
        case ROPE_HALVES: paged_append_kernel<T, 1, ROPE_HALVES, C><<<grid, threads, 0, st>>>(a); break;
        case ROPE_HALVES_LANE: paged_append_kernel<T, 2, ROPE_HALVES_LANE, C><<<grid, threads, 0, st>>>(a); break;
        default: paged_append_kernel<T, VPL, ROPE_HALVES_SMEM, C><<<grid, threads, smem, st>>>(a); break;
    }
    return check_launch("paged_append_kernel");
}

// A call's arguments beside the cache and the batch, as the ABI has them.
struct AppendCall {
    const void* q;
    int64_t q_token, q_head, n_heads;
    const void* k;
    int64_t k_token, k_head;
    const void* v;
    int64_t v_token, v_head;
    const void *q_weight, *k_weight;
    int weight_dtype;
    float eps;
    const float* rope;
    int64_t n_pos, rotary_dim;
    int interleaved;
    const int32_t* positions;
    void* q_out;
    int64_t out_token, out_head;
    int32_t* status;
};

// Checks them for a cache of `dims` and vectors of dims.dtype, and fills *a but for the pages;
// *vpl = 0: there is nothing to do.
hmm_status_t plan_append(const AppendCall& c, const hmm_paged_cache_t& dims, const hmm_paged_batch_t* batch, bool quant,
                         AppendArgs* a, int* mode, int* vpl);

}  // namespace serve
}  // namespace hmm
