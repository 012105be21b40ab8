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
    FastDiv by_group;
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
        const int phys = page_of(a, s, key / a.page_tokens);
        if (phys < 0) continue;
        const int in = key % a.page_tokens;
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

// Joins (maximum, sum, row) pieces of up to 16 rows, which several warps or CTAs summed
// over different keys, in their order, and writes the rows out; rows that come out not
// finite are computed again by attn_row_exact.  piece(i, row, -1 / -2 / d) reads the
// maximum, sum or value of piece i; `share` holds 16 x pieces floats.  Whole block.
template <typename T, typename Piece>
__device__ __forceinline__ void finish_rows(const AttnArgs& a, int s, const Seq& q, int kvh, int row0,
                                            int rows, int pieces, Piece piece, float* share, int* again) {
    if (threadIdx.x == 0) *again = 0;
    const int lane = threadIdx.x & 31;
    // each piece's share of the row: exp2(m_i - m) / sum_k exp2(m_k - m) l_k
    for (int r = threadIdx.x >> 5; r < rows; r += blockDim.x >> 5) {
        float m = -INFINITY, l = 0.0f;
        for (int p = lane; p < pieces; p += 32) m = fmaxf(m, piece(p, r, -1));
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
        const float ms = m == -INFINITY ? 0.0f : m;
        for (int p = lane; p < pieces; p += 32) {
            const float wgt = ex2(piece(p, r, -1) - ms);
            share[r * pieces + p] = wgt;
            if (wgt != 0.0f) l = fmaf(wgt, piece(p, r, -2), l);
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
        const float inv = l == 0.0f ? 0.0f : 1.0f / l;
        __syncwarp();
        for (int p = lane; p < pieces; p += 32) {
            const float wgt = share[r * pieces + p];
            share[r * pieces + p] = wgt == 0.0f ? 0.0f : wgt * inv;   // (0: a piece in which the row saw nothing)
        }
        if (lane == 0) {
            if (l != l) atomicOr(again, 1 << r);
            if (a.lse) {
                const int tok = a.by_group(row0 + r);
                a.lse[(int64_t)(q.begin + tok) * a.hq + kvh * a.group + row0 + r - tok * a.group] =
                    l == 0.0f ? -INFINITY : (m + log2f(l)) * LN2;
            }
        }
    }
    __syncthreads();
    const int pairs = a.D / 2;
    for (int i = threadIdx.x; i < rows * pairs; i += blockDim.x) {
        const int r = i / pairs, d = 2 * (i - r * pairs);
        float x = 0.0f, y = 0.0f;
#pragma unroll 4
        for (int p = 0; p < pieces; ++p) {
            const float wgt = share[r * pieces + p];
            const float u = piece(p, r, d), v = piece(p, r, d + 1);
            x = wgt == 0.0f ? x : fmaf(wgt, u, x);
            y = wgt == 0.0f ? y : fmaf(wgt, v, y);
        }
        if (!isfinite(x) || !isfinite(y)) atomicOr(again, 1 << r);
        const int tok = a.by_group(row0 + r), head = kvh * a.group + row0 + r - tok * a.group;
        *reinterpret_cast<uint32_t*>(a.out + 2 * (((int64_t)(q.begin + tok) * a.hq + head) * a.D + d)) =
            pack2<T>(x, y);
    }
    __syncthreads();
    const int bits = *again;
    for (int r = threadIdx.x >> 5; r < rows; r += blockDim.x >> 5)
        if ((bits >> r) & 1) attn_row_exact<T>(a, s, q, kvh, row0 + r);
    __syncthreads();
}

// Launches a kernel that begins with griddepcontrol.wait: its blocks may be set up while
// the kernel before it on the stream still runs.
template <typename F, typename A>
hmm_status_t launch_behind(F fn, dim3 grid, int threads, size_t smem, cudaStream_t st, const A& args,
                           const char* what) {
    cudaLaunchConfig_t c{};
    c.gridDim = grid;
    c.blockDim = dim3(threads);
    c.dynamicSmemBytes = smem;
    c.stream = st;
    cudaLaunchAttribute at{};
    at.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at.val.programmaticStreamSerializationAllowed = 1;
    c.attrs = &at;
    c.numAttrs = 1;
    HMM_CUDA_TRY(cudaLaunchKernelEx(&c, fn, args));
    return check_launch(what);
}

}  // namespace serve
}  // namespace hmm
