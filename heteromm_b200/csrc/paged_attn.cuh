// paged_attn.cuh — what the two attention kernels over a paged cache share: the
// arguments, which keys a row sees, and a row computed from the definition.
//
//   o = sum_i p_i v_i / sum_i p_i,  p_i = exp(scale q.k_i - m),  m = the largest score
//   key i is seen from position p iff i < kv_len, (not causal or i <= p) and
//   (no window or i > p - window or i < sinks)
#pragma once

#include "paged_serve.cuh"

namespace hmm {
namespace serve {

// n / d for 0 <= n < 2^31 by a multiplication: mul = floor(2^(31 + s) / d) + 1 with 2^s
// the power of two at or above d.
struct FastDiv {
    uint32_t mul;
    int shift;
    __host__ static FastDiv of(int d) {
        int s = 0;
        while ((int64_t(1) << s) < d) ++s;
        if (s == 0) return FastDiv{0, 0};
        return FastDiv{(uint32_t)((uint64_t(1) << (31 + s)) / (uint64_t)d + 1), s - 1};
    }
    __device__ __forceinline__ int operator()(int n) const {
        return mul == 0 ? n : (int)(__umulhi((uint32_t)n, mul) >> shift);
    }
};

struct AttnArgs {
    Batch b;
    Pages k, v;
    const unsigned char* q;      // token / head strides in bytes
    int64_t q_token, q_head;
    unsigned char* out;          // [n_tokens][hq][D], contiguous
    float* lse;                  // [n_tokens][hq] or null
    float scale, scale_log2;     // scale * log2(e)
    int causal, window, sinks;
    int hq, hk, group, D, page_tokens, n_pages;
    FastDiv by_group, by_page;   // n / group, key / page_tokens
    int64_t max_kv;
    int32_t* status;
};

// A row of a unit (sequence, KV head): row r is new token r / group, head r % group.
struct Span {                    // keys [0, sink) and [lo, hi) hold all that some row of a tile sees
    int p0, p1;                  // positions of the tile's first and last row
    int lo, hi, sink;
};

// -1 for a row before the first cached token: it sees nothing.
__device__ __forceinline__ int row_pos(const AttnArgs& a, const Seq& q, int row) {
    return max(-1, q.kv - q.n_new + a.by_group(row));
}

__device__ __forceinline__ Span tile_span(const AttnArgs& a, const Seq& q, int row0, int row1) {
    Span s;
    s.p0 = row_pos(a, q, row0);
    s.p1 = row_pos(a, q, row1 - 1);
    s.hi = a.causal ? max(0, min(q.kv, s.p1 + 1)) : q.kv;
    s.lo = a.window > 0 ? min(s.hi, max(0, s.p0 - a.window + 1)) : 0;
    s.sink = a.window > 0 ? min(a.sinks, s.lo) : 0;
    return s;
}

__device__ __forceinline__ bool span_has(const Span& s, int key) {
    return key < s.sink || (key >= s.lo && key < s.hi);
}

__device__ __forceinline__ bool sees(const AttnArgs& a, int kv, int pos, int key) {
    return key < kv && (!a.causal || key <= pos) &&
           (a.window <= 0 || key > pos - a.window || key < a.sinks);
}

// The physical page of a token, or -1 with HMM_STATUS_PAGE_BOUNDS set.
__device__ __forceinline__ int page_of(const AttnArgs& a, int s, int logical) {
    const int e = __ldg(a.b.table + (int64_t)s * a.b.pages_per_seq + logical);
    if (e >= 0 && e < a.n_pages) return e;
    atomicOr(a.status, HMM_STATUS_PAGE_BOUNDS);
    return -1;
}

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

constexpr float LN2 = 0.693147180559945309417f;

// One row from the definition, by one warp, key by key in fp32: the row's
// result where the tiled product does not hold.  A tile multiplies weights of
// zero with the values of keys that only other rows see, and a zero times an
// infinity or NaN there is NaN; such a row comes here, so that what a row does
// not see never reaches it.  (It also comes here, to the same NaN or infinity,
// when what it sees is not finite.)
template <typename T>
__device__ __forceinline__ void attn_row_exact(const AttnArgs& a, int s, const Seq q, int kvh, int row) {
    constexpr int NV = 8;   // 32 lanes x 8 = D <= 256
    const int lane = threadIdx.x & 31;
    const int tok = q.begin + row / a.group, head = kvh * a.group + row % a.group;
    const int pos = row_pos(a, q, row);
    const Span sp = tile_span(a, q, row, row + 1);
    const T* qr = reinterpret_cast<const T*>(a.q + tok * a.q_token + head * a.q_head);
    float qf[NV], acc[NV], m = -INFINITY, l = 0.0f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        qf[i] = lane + 32 * i < a.D ? to_f32<T>(qr[lane + 32 * i]) : 0.0f;
        acc[i] = 0.0f;
    }
    for (int key = sp.sink > 0 ? 0 : sp.lo; key < sp.hi; ++key) {
        if (key == sp.sink && key < sp.lo) key = sp.lo;
        if (key >= sp.hi) break;
        if (!sees(a, q.kv, pos, key)) continue;
        const int lp = a.by_page(key), phys = page_of(a, s, lp);
        if (phys < 0) continue;
        const int in = key - lp * a.page_tokens;
        const T* kr = reinterpret_cast<const T*>(a.k.base + phys * a.k.page + kvh * a.k.head + in * a.k.token);
        const T* vr = reinterpret_cast<const T*>(a.v.base + phys * a.v.page + kvh * a.v.head + in * a.v.token);
        float x = 0.0f;
#pragma unroll
        for (int i = 0; i < NV; ++i)
            if (lane + 32 * i < a.D) x = fmaf(qf[i], to_f32<T>(kr[lane + 32 * i]), x);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
        x *= a.scale_log2;
        const float mn = fmaxf(m, x), ms = mn == -INFINITY ? 0.0f : mn;
        const float al = ex2(m - ms), p = ex2(x - ms);
        l = l * al + p;
        m = mn;
#pragma unroll
        for (int i = 0; i < NV; ++i)
            if (lane + 32 * i < a.D) acc[i] = acc[i] * al + p * to_f32<T>(vr[lane + 32 * i]);
    }
    T* o = reinterpret_cast<T*>(a.out) + ((int64_t)tok * a.hq + head) * a.D;
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll
    for (int i = 0; i < NV; ++i)
        if (lane + 32 * i < a.D) o[lane + 32 * i] = l == 0.0f ? T(0.0f) : T(acc[i] * inv);
    if (a.lse && lane == 0)
        a.lse[(int64_t)tok * a.hq + head] = l == 0.0f ? -INFINITY : (m + log2f(l)) * LN2;
}

// The joined rows' values: K quads a thread and P pieces at a time, K * P reads in flight.
template <typename T, int K, int P, typename Value>
__device__ __forceinline__ void join_values(const AttnArgs& a, const Seq& q, int kvh, int row0, int rows, int pieces,
                                            Value value, const float* top, int* again) {
    const int quads = a.D / 4, all = rows * quads;
    for (int i0 = threadIdx.x; i0 < all; i0 += K * blockDim.x) {
        float4 x[K];
        int row[K], col[K];
#pragma unroll
        for (int k = 0; k < K; ++k) {
            const int i = min(i0 + k * (int)blockDim.x, all - 1);
            row[k] = i / quads;
            col[k] = i - row[k] * quads;
            x[k] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        }
        for (int p0 = 0; p0 < pieces; p0 += P) {
            float4 v[K][P];
#pragma unroll
            for (int k = 0; k < K; ++k)
#pragma unroll
                for (int p = 0; p < P; ++p) v[k][p] = value(min(p0 + p, pieces - 1), row[k], col[k]);
#pragma unroll
            for (int k = 0; k < K; ++k)
#pragma unroll
                for (int p = 0; p < P; ++p) {
                    const float w = p0 + p < pieces ? top[row[k] * pieces + p0 + p] : 0.0f;
                    if (w != 0.0f) {
                        x[k].x = fmaf(w, v[k][p].x, x[k].x); x[k].y = fmaf(w, v[k][p].y, x[k].y);
                        x[k].z = fmaf(w, v[k][p].z, x[k].z); x[k].w = fmaf(w, v[k][p].w, x[k].w);
                    }
                }
        }
#pragma unroll
        for (int k = 0; k < K; ++k) {
            if (i0 + k * (int)blockDim.x >= all) continue;
            if (!isfinite(x[k].x) || !isfinite(x[k].y) || !isfinite(x[k].z) || !isfinite(x[k].w))
                atomicOr(again, 1 << row[k]);
            const int tok = a.by_group(row0 + row[k]), head = kvh * a.group + row0 + row[k] - tok * a.group;
            *reinterpret_cast<uint2*>(a.out + 2 * (((int64_t)(q.begin + tok) * a.hq + head) * a.D + 4 * col[k])) =
                make_uint2(pack2<T>(x[k].x, x[k].y), pack2<T>(x[k].z, x[k].w));
        }
    }
}

// Joins (maximum, sum, row) pieces of up to 16 rows, which several warps or CTAs summed
// over different keys, in their order, and writes the rows out; rows that come out not
// finite are computed again by attn_row_exact.  stat(i, row, k) reads piece i's maximum
// (k = 0) or sum (1), value(i, row, c) its columns 4 c ... 4 c + 3; `share` holds
// 32 x pieces floats.  A piece with a score of NaN or +inf has a maximum of +inf (and no
// other has: a sum with it is NaN).  Whole block, 128 threads.  FAR: the pieces lie in memory, many of
// them maybe, and their reads' latency is what it costs (one token over 4,000, 31 pieces:
// the call took 25 us with two at a time, 17 with eight; sixteen gave no more).
template <typename T, bool FAR, typename Stat, typename Value>
__device__ __forceinline__ void finish_rows(const AttnArgs& a, int s, const Seq& q, int kvh, int row0,
                                            int rows, int pieces, Stat stat, Value value, float* share,
                                            int* again) {
    if (threadIdx.x == 0) *again = 0;
    float* top = share;                 // [row][piece] maxima, then the pieces' shares of the row
    float* sum = share + 16 * pieces;
#pragma unroll 4
    for (int i = threadIdx.x; i < rows * pieces; i += blockDim.x) {
        const int r = i / pieces, p = i - r * pieces;
        top[i] = stat(p, r, 0);
        sum[i] = stat(p, r, 1);
    }
    __syncthreads();
    // exp2(m_i - m) / sum_k exp2(m_k - m) l_k, eight threads a row
    {
        const int r = threadIdx.x >> 3, t = threadIdx.x & 7;
        const bool live = r < rows;
        float m = -INFINITY, l = 0.0f;
        for (int p = t; live && p < pieces; p += 8) m = fmaxf(m, top[r * pieces + p]);
#pragma unroll
        for (int o = 4; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
        const float ms = m == -INFINITY ? 0.0f : m;
        for (int p = t; live && p < pieces; p += 8) {
            const float w = ex2(top[r * pieces + p] - ms);
            top[r * pieces + p] = w;
            if (w != 0.0f) l = fmaf(w, sum[r * pieces + p], l);   // (0: nothing seen in the piece, or nothing beside the others)
        }
#pragma unroll
        for (int o = 4; o > 0; o >>= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
        const float inv = l == 0.0f ? 0.0f : 1.0f / l;
        for (int p = t; live && p < pieces; p += 8) {
            const float w = top[r * pieces + p];
            top[r * pieces + p] = w == 0.0f ? 0.0f : w * inv;
        }
        if (live && t == 0) {
            if (l != l) atomicOr(again, 1 << r);
            if (a.lse) {
                const int tok = a.by_group(row0 + r);
                a.lse[(int64_t)(q.begin + tok) * a.hq + kvh * a.group + row0 + r - tok * a.group] =
                    l == 0.0f ? -INFINITY : (m + log2f(l)) * LN2;
            }
        }
    }
    __syncthreads();
    if (FAR && rows * (a.D / 4) <= (int)blockDim.x)
        join_values<T, 1, 8>(a, q, kvh, row0, rows, pieces, value, top, again);
    else
        join_values<T, 4, 2>(a, q, kvh, row0, rows, pieces, value, top, again);
    __syncthreads();
    const int bits = *again;
    for (int r = threadIdx.x >> 5; r < rows; r += blockDim.x >> 5)
        if ((bits >> r) & 1) attn_row_exact<T>(a, s, q, kvh, row0 + r);
    __syncthreads();
}

// Launches a kernel; with `behind` its blocks may start while the kernel before it on the
// stream, which lets them (griddepcontrol.launch_dependents), still runs.
template <typename... P, typename... A>
hmm_status_t launch(void (*fn)(P...), dim3 grid, int threads, size_t smem, bool behind, cudaStream_t st,
                    const char* what, const A&... args) {
    cudaLaunchConfig_t c{};
    c.gridDim = grid;
    c.blockDim = dim3(threads);
    c.dynamicSmemBytes = smem;
    c.stream = st;
    cudaLaunchAttribute at{};
    at.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at.val.programmaticStreamSerializationAllowed = 1;
    c.attrs = &at;
    c.numAttrs = behind ? 1 : 0;
    HMM_CUDA_TRY(cudaLaunchKernelEx(&c, fn, args...));
    return check_launch(what);
}

}  // namespace serve
}  // namespace hmm
