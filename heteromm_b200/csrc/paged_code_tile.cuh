// paged_code_tile.cuh — what the rows kernel does with a warp's tile of 32 keys of a cache in 8
// bits: copies of its codes, scores, the product with V.
//
// The products are taken in fp16, whatever q is: it holds every code times its scale, and one
// instruction makes two of two e4m3 codes (2.2 clocks a scheduler measured; to bf16 it takes six
// of 2).  bf16 queries go to fp16 times a power of two per row.
//
// Codes come as TMA boxes of a page's rows, 128 bytes (D = 64: 64) wide and swizzled over as
// many, scale bytes by one 16-byte cp.async a lane (as bulk copies they doubled the requests;
// codes by cp.async too are held by what the L1 cache keeps in flight).
//
// MMA m16n8k16: lane = 4 n + c holds key n's (K) or column n's (V) values 2 c, 2 c + 1, + 8.
//   K: a lane takes the values in the order of its codes, 16 or 32 of a row in a run, four a step:
//      queries are laid out alike (code_of_step).
//   V: lane n takes columns [W n, W n + W), W = D / 8, a block of eight columns being the i-th of
//      all lanes: 16 codes of a row in a read, one scale group a lane.
#pragma once

#include "paged_attn.cuh"

namespace hmm {
namespace serve {

constexpr int CT_KEYS = 32;

__device__ __forceinline__ void cp16(uint32_t dst, const void* src, bool real) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(real ? 16 : 0)
                 : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// The first of the four codes that step k of a key's product takes in lane c of four.
template <int DP>
__device__ __forceinline__ int code_of_step(int k, int c) {
    return DP == 64 ? 16 * c + 4 * k : (k >> 3) * 128 + 32 * c + 4 * (k & 7);
}

// Byte of 16-byte piece p of row r in a tile.
template <int DP>
__device__ __forceinline__ int code_at(int r, int p) {
    if (DP == 64) return r * 64 + ((p ^ (r >> 1 & 3)) * 16);
    return (p >> 3) * (CT_KEYS * 128) + r * 128 + (((p & 7) ^ (r & 7)) * 16);
}

// Pairs of codes to fp16, unscaled, of a word [a0, b0, a1, b1]: (a0, b0) and (a1, b1).
// int8: 4 + (n + 128) / 256 less 4.5, n / 256.
template <int C>
__device__ __forceinline__ void code_pairs(uint32_t w, uint32_t& a, uint32_t& b) {
    if (C == CODEC_E4M3) {
        asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, l;\n\tcvt.rn.f16x2.e4m3x2 %1, h;\n\t}"
            : "=r"(a), "=r"(b)
            : "r"(w));
    } else {
        const uint32_t x = w ^ 0x80808080u;
        asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(a) : "r"(__byte_perm(x, 0x44u, 0x4140)), "r"(0x44804480u));
        asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(b) : "r"(__byte_perm(x, 0x44u, 0x4342)), "r"(0x44804480u));
    }
}
// The factors of two scale bytes as a pair: an infinity for 255, which makes NaN of codes of zero.
template <int C>
__device__ __forceinline__ uint32_t code_factors(uint32_t a, uint32_t b) {
    constexpr uint32_t UP = C == CODEC_E4M3 ? 0u : 8u << 23;      // (int8: of n / 256)
    uint32_t d;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(d) : "f"(__uint_as_float(min((b << 23) + UP, 0x7f800000u))),
        "f"(__uint_as_float(min((a << 23) + UP, 0x7f800000u))));
    return d;
}

__device__ __forceinline__ void mma_half(float* d, const uint32_t* a, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// A row of q (null: zeros), half h of the fragments.  bf16 values go to fp16 times the power of two that
// brings the row's largest finite one to 2^14 ... 2^15: exact down to 2^-28 of it, and off by
// 2^-39 of it below (half a step of fp16's subnormal numbers, 2^-25, beside 2^14).  Returns what the row's scores are times then.  Lanes of a row: 4 n + c.
template <typename T, int DP>
__device__ __forceinline__ float code_queries(const unsigned char* src, int D, int h, uint32_t (*qf)[4]) {
    const int c = threadIdx.x & 3;
    uint32_t top = 0;
#pragma unroll
    for (int k = 0; k < DP / 16; ++k) {
        const int d = code_of_step<DP>(k, c);
        const uint2 x = src && d < D ? __ldg(reinterpret_cast<const uint2*>(src + 2 * d)) : make_uint2(0u, 0u);
        qf[k][h] = x.x;
        qf[k][h + 2] = x.y;
        if (!std::is_same<T, __half>::value) {
            const uint32_t m[4] = {x.x & 0x7fffu, x.x >> 16 & 0x7fffu, x.y & 0x7fffu, x.y >> 16 & 0x7fffu};
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (m[j] < 0x7f80u) top = max(top, m[j]);
        }
    }
    if (std::is_same<T, __half>::value) return 1.0f;
    top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
    top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
    const int e = max((int)(top >> 7), 15);       // the largest's biased exponent
    const float up = __uint_as_float((uint32_t)(127 + 14 + 127 - e) << 23);
#pragma unroll
    for (int k = 0; k < DP / 16; ++k)
#pragma unroll
        for (int j = 0; j < 4; j += 2) {
            const float2 f = unpack2<T>(qf[k][h + j]);
            qf[k][h + j] = pack2<__half>(f.x * up, f.y * up);
        }
    return __uint_as_float((uint32_t)(e - 14) << 23);
}

// Copies of a tile's scale bytes, K's by the lower lanes of a warp and V's by the upper ones, 16 bytes
// each.  A lane's are always of the same box, so that it holds where in a page they begin.
struct ScaleCopy {
    const unsigned char* base;
    int64_t page;
    int box, dst;        // (box < 0: none for this lane)
};
__device__ __forceinline__ ScaleCopy scale_copy(const AttnArgs& a, int kvh, int box_rows, int v_scales) {
    const int lane = threadIdx.x & 31, per = a.quant.per_token, at = 16 * (lane & 15), bytes = box_rows * per;
    const Pages& x = lane < 16 ? a.k : a.v;
    const int box = at / bytes;                                  // (a box's bytes are a multiple of 16)
    return ScaleCopy{x.base + kvh * x.head + a.quant.scales + at - box * bytes, x.page, at < CT_KEYS * per ? box : -1,
                     (lane < 16 ? 0 : v_scales) + at};
}
// Lane s holds (page, row) of box s; a page of n_pages is out of range.
__device__ __forceinline__ void code_copy_scales(const AttnArgs& a, const ScaleCopy& c, int page, int row, uint32_t dst) {
    const int pg = __shfl_sync(0xffffffffu, page, c.box & 31), rw = __shfl_sync(0xffffffffu, row, c.box & 31);
    const bool real = pg < a.n_pages;   // (else zeros, as the codes')
    if (c.box >= 0) cp16(dst + c.dst, real ? c.base + pg * c.page + (int64_t)rw * a.quant.per_token : c.base, real);
}

// Scores of 16 rows and 32 keys.  (Four sums at a time: an MMA waits for the one before it in its own.)
template <int DP, int C>
__device__ __forceinline__ void code_scores(const unsigned char* k, const unsigned char* scales, int per,
                                            const uint4* qs, float (*sc)[4]) {
    constexpr int PIECES = DP == 64 ? 1 : 2;
    const int lane = threadIdx.x & 31, n = lane >> 2, c = lane & 3;
#pragma unroll
    for (int h = 0; h < (DP + 127) / 128; ++h) {
        uint32_t m[4];
#pragma unroll
        for (int nb = 0; nb < 4; ++nb) {
            const uint32_t s = scales[(8 * nb + n) * per + min(DP == 64 ? c >> 1 : 4 * h + c, per - 1)];
            m[nb] = code_factors<C>(s, s);
        }
#pragma unroll
        for (int y = 0; y < PIECES; ++y) {
            uint4 w[4];
#pragma unroll
            for (int nb = 0; nb < 4; ++nb)
                w[nb] = *reinterpret_cast<const uint4*>(k + code_at<DP>(8 * nb + n, DP == 64 ? c : 8 * h + 2 * c + y));
#pragma unroll
            for (int z = 0; z < 4; ++z) {
                const uint4 qv = qs[((h * PIECES + y) * 4 + z) * 32 + lane];
                const uint32_t qa[4] = {qv.x, qv.y, qv.z, qv.w};
#pragma unroll
                for (int nb = 0; nb < 4; ++nb) {
                    const uint32_t u = z == 0 ? w[nb].x : z == 1 ? w[nb].y : z == 2 ? w[nb].z : w[nb].w;
                    uint32_t b0, b1;
                    code_pairs<C>(u, b0, b1);
                    mma_half(sc[nb], qa, mul_pair<__half>(b0, m[nb]), mul_pair<__half>(b1, m[nb]));
                }
            }
        }
    }
}

// o += p V over 32 keys; p [2][4] fragments of 16 keys.
template <int DP, int C>
__device__ __forceinline__ void code_product(const unsigned char* v, const unsigned char* scales, int per,
                                             const uint32_t* p, float (*o)[4]) {
    constexpr int W = DP / 8, READS = DP == 256 ? 2 : 1;         // columns of a lane, 16-byte reads of a row
    const int lane = threadIdx.x & 31, n = lane >> 2, c = lane & 3, group = min(W * n / Q_GROUP, per - 1);
#pragma unroll
    for (int x = 0; x < 2; ++x) {
        const int r = 16 * x + 2 * c;                            // keys r, r + 1, r + 8, r + 9
        const unsigned char* s = scales + r * per + group;
        const uint32_t f0 = code_factors<C>(s[0], s[per]), f1 = code_factors<C>(s[8 * per], s[9 * per]);
#pragma unroll
        for (int y = 0; y < READS; ++y) {
            uint32_t w[4][4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const unsigned char* src = v + code_at<DP>(r + (i & 1) + 8 * (i >> 1), DP == 64 ? n >> 1 : READS * n + y);
                if (DP == 64) {
                    const uint2 t = *reinterpret_cast<const uint2*>(src + 8 * (n & 1));
                    w[i][0] = t.x;
                    w[i][1] = t.y;
                } else {
                    const uint4 t = *reinterpret_cast<const uint4*>(src);
                    w[i][0] = t.x;
                    w[i][1] = t.y;
                    w[i][2] = t.z;
                    w[i][3] = t.w;
                }
            }
#pragma unroll
            for (int t = 0; t < (DP == 64 ? 2 : 4); ++t)
#pragma unroll
                for (int h = 0; h < 2; ++h) {                    // codes 2 h, 2 h + 1 of the words
                    uint32_t a0, a1, b0, b1;
                    code_pairs<C>(__byte_perm(w[0][t], w[1][t], h ? 0x7362 : 0x5140), a0, a1);
                    code_pairs<C>(__byte_perm(w[2][t], w[3][t], h ? 0x7362 : 0x5140), b0, b1);
                    const int i = 16 * y + 4 * t + 2 * h;
                    mma_half(o[i], p + 4 * x, mul_pair<__half>(a0, f0), mul_pair<__half>(b0, f1));
                    mma_half(o[i + 1], p + 4 * x, mul_pair<__half>(a1, f0), mul_pair<__half>(b1, f1));
                }
        }
    }
}

// Row half h of o to a row of `dst` (16-byte aligned): lane c has columns [2 c W, 2 c W + 2 W).
template <int DP>
__device__ __forceinline__ void code_row(const float (*o)[4], int h, float* dst) {
    constexpr int W = DP / 8;
    dst += 2 * W * (threadIdx.x & 3);
#pragma unroll
    for (int e = 0; e < 2; ++e)
#pragma unroll
        for (int i = 0; i < W; i += 4)
            *reinterpret_cast<float4*>(dst + e * W + i) =
                make_float4(o[i][2 * h + e], o[i + 1][2 * h + e], o[i + 2][2 * h + e], o[i + 3][2 * h + e]);
}

}  // namespace serve
}  // namespace hmm
