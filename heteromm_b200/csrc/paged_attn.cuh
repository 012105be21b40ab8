// paged_attn.cuh — what the two attention kernels over a paged cache share: the
// arguments, which keys a row sees, and a row computed from the definition.
//
//   o = sum_i p_i v_i / sum_i p_i,  p_i = exp(scale q.k_i - m),  m = the largest score
//   key i is seen from position p iff i < kv_len, (not causal or i <= p) and
//   (no window or i > p - window or i < sinks)
#pragma once

#include <float.h>

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

// A key's K and V rows; null if its page is flagged.
struct KeyRows {
    const unsigned char *k, *v;
};
__device__ __forceinline__ KeyRows key_rows(const AttnArgs& a, int s, int kvh, int key) {
    const int lp = a.by_page(key), phys = page_of(a, s, lp), in = key - lp * a.page_tokens;
    if (phys < 0) return KeyRows{nullptr, nullptr};
    return KeyRows{a.k.base + phys * a.k.page + kvh * a.k.head + in * a.k.token,
                   a.v.base + phys * a.v.page + kvh * a.v.head + in * a.v.token};
}

template <typename T>
__device__ __forceinline__ void unpack8(const uint4& w, float* f) {
    const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 p = unpack2<T>(u[i]);
        f[2 * i] = p.x;
        f[2 * i + 1] = p.y;
    }
}

// Whether one of eight values is an infinity or NaN: all bits of its exponent.
template <typename T>
__device__ __forceinline__ bool any_not_finite(const uint4& w) {
    constexpr uint32_t E = std::is_same<T, __half>::value ? 0x7c007c00u : 0x7f807f80u;
    return (__vcmpeq2(w.x & E, E) | __vcmpeq2(w.y & E, E) | __vcmpeq2(w.z & E, E) | __vcmpeq2(w.w & E, E)) != 0u;
}

// The columns that came out not finite of rows row0 + i, bit i of `rows`, from the
// definition, by one warp in fp32: what the tiled product cannot tell.  A tile multiplies
// weights of zero with the values of keys that only other rows see, and a zero times an
// infinity or NaN there is NaN; such rows come here, so that what a row does not see never
// reaches it.  Their scores are finite or, all but one, -inf, and their other columns and
// lse stand.  (A row whose columns are finite is passed over, and one with a NaN score,
// whose columns are NaN, stays so.)
//
// First the values alone: a seen NaN decides its column, as do infinities of both signs, and
// a product that is infinite is right if the row sees an infinity (an unseen one gives NaN).
// The keys that all the rows see are gone through once.  So one bad value that many rows see
// costs each little.  What is left is added up again, row by row: a lane scores one of 32
// keys, and groups of lanes, eight columns each, add values.
//
// 4,096 tokens, 32/8 heads of 128, one NaN or infinity: 0.36 ms if the first key holds it, 0.9
// in the middle (row by row and key by key 227 and 180; without it 0.15).  One that some rows
// of a unit see and others do not, the last key's: 16 ms.
// U: loops are unrolled so far.  The code is never reached as a rule, but its size is felt by
// kernels that stream (the decode batch 351 -> 355 us with 16 in the join; 352 with 1).
template <typename T, int U>
__device__ __forceinline__ void attn_rows_exact(const AttnArgs& a, int s, const Seq q, int kvh, int row0, unsigned rows) {
    const int lane = threadIdx.x & 31, vecs = a.D / 8;
    const int lanes = vecs > 1 ? 2 << (31 - __clz(vecs - 1)) : 1, groups = 32 / lanes;   // of a V row
    const int gl = lane & (lanes - 1), group = lane / lanes;
    auto result = [&](int i) {   // the lane's columns of row row0 + i
        const int r = row0 + i, tok = a.by_group(r);
        return a.out + 2 * (((int64_t)(q.begin + tok) * a.hq + kvh * a.group + r - tok * a.group) * a.D + 8 * gl);
    };
    auto bad_columns = [&](int i, uint32_t* nan, uint32_t* inf) {   // a bit per column
        float f[8];
        unpack8<T>(gl < vecs ? *reinterpret_cast<const uint4*>(result(i)) : make_uint4(0u, 0u, 0u, 0u), f);
        *nan = *inf = 0;
#pragma unroll
        for (int c = 0; c < 8; ++c) {
            *nan |= (f[c] != f[c] ? 1u : 0u) << c;
            *inf |= (isinf(f[c]) ? 1u : 0u) << c;
        }
    };
    auto values = [&](const unsigned char* v, int i) {   // of the i-th of a group's `lanes` keys
        const unsigned char* p = reinterpret_cast<const unsigned char*>(
            __shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(v), i * groups + group));
        return p && gl < vecs ? __ldg(reinterpret_cast<const uint4*>(p) + gl) : make_uint4(0u, 0u, 0u, 0u);
    };
    auto rows_of = [&](int key, int end) { return key < end ? key_rows(a, s, kvh, key) : KeyRows{nullptr, nullptr}; };
    uint32_t met = 0;   // NaN, inf, -inf seen in the lane's columns, a byte each
    auto met_nan = [&] { return (met | (met >> 8 & met >> 16)) & 0xffu; };
    auto undecided = [&](uint32_t nan, uint32_t inf) { return (nan | (inf & ~(met >> 8 | met >> 16))) & ~met_nan(); };
    auto scan = [&](int k0, int k1, uint32_t nan, uint32_t inf) {   // keys [k0, k1), until the columns are decided
        if (k0 >= k1 || !__any_sync(0xffffffffu, undecided(nan, inf) != 0)) return;
        KeyRows r = rows_of(k0 + lane, k1);
        for (; k0 < k1; k0 += 32) {
            const KeyRows next = rows_of(k0 + 32 + lane, k1);
#pragma unroll U
            for (int i = 0; i < lanes; ++i) {
                const uint4 w = values(r.v, i);
                if (any_not_finite<T>(w)) {
                    float f[8];
                    unpack8<T>(w, f);
#pragma unroll
                    for (int c = 0; c < 8; ++c)
                        met |= (f[c] != f[c] ? 1u : f[c] == INFINITY ? 0x100u : f[c] == -INFINITY ? 0x10000u : 0u) << c;
                }
            }
            r = next;
            for (int w = lanes; w < 32; w <<= 1) met |= __shfl_xor_sync(0xffffffffu, met, w);
            if (!__any_sync(0xffffffffu, undecided(nan, inf) != 0)) break;
        }
    };
    if (rows == 0) return;
    // the keys [all0, all1) that all of them see
    const int first = row0 + __ffs(rows) - 1, last = row0 + 31 - __clz(rows);
    const int all0 = tile_span(a, q, last, last + 1).lo, all1 = max(all0, tile_span(a, q, first, first + 1).hi);
    {
        uint32_t nan = 0, inf = 0;
        for (unsigned left = rows; left; left &= left - 1) {
            uint32_t n, f;
            bad_columns(__ffs(left) - 1, &n, &f);
            nan |= n;
            inf |= f;
        }
        scan(all0, all1, nan, inf);
    }
    const uint32_t met_all = met;
    for (; rows; rows &= rows - 1) {
        const int i = __ffs(rows) - 1, row = row0 + i;
        const Span sp = tile_span(a, q, row, row + 1);   // all of it is seen
        uint32_t nan, inf;
        bad_columns(i, &nan, &inf);
        met = met_all;
#pragma unroll 1
        for (int part = 0; part < 3; ++part)             // first tokens; behind and before the common ones
            scan(part == 0 ? 0 : part == 1 ? sp.lo : max(all1, sp.lo),
                 part == 0 ? sp.sink : part == 1 ? min(all0, sp.hi) : sp.hi, nan, inf);
        const uint32_t left = undecided(nan, inf), is_nan = met_nan() & (nan | inf);
        float acc[8], m = -INFINITY, l = 0.0f;
#pragma unroll
        for (int c = 0; c < 8; ++c) acc[c] = 0.0f;
        if (__any_sync(0xffffffffu, left != 0)) {
            const int tok = a.by_group(row), n = sp.sink + sp.hi - sp.lo;
            const uint4* qr = reinterpret_cast<const uint4*>(a.q + (q.begin + tok) * a.q_token +
                                                             (kvh * a.group + row - tok * a.group) * a.q_head);
            for (int i0 = 0; i0 < n; i0 += 32) {
                const int at = i0 + lane;
                const KeyRows r = rows_of(at < sp.sink ? at : sp.lo + at - sp.sink, at < n ? INT32_MAX : 0);
                float x = -INFINITY;
                if (r.k) {
                    x = 0.0f;
#pragma unroll U < 8 ? U : 8
                    for (int c = 0; c < vecs; ++c) {
                        float kf[8], qf[8];
                        unpack8<T>(__ldg(reinterpret_cast<const uint4*>(r.k) + c), kf);
                        unpack8<T>(__ldg(qr + c), qf);
#pragma unroll
                        for (int e = 0; e < 8; ++e) x = fmaf(qf[e], kf[e], x);
                    }
                    x *= a.scale_log2;
                }
                float mn = fmaxf(m, x);
#pragma unroll
                for (int w = 16; w > 0; w >>= 1) mn = fmaxf(mn, __shfl_xor_sync(0xffffffffu, mn, w));
                const float ms = mn == -INFINITY ? 0.0f : mn, al = ex2(m - ms), p = ex2(x - ms);
                l = fmaf(l, al, p);                      // (a lane's share)
                m = mn;
#pragma unroll
                for (int c = 0; c < 8; ++c) acc[c] = isinf(acc[c]) ? acc[c] : acc[c] * al;
                // (a weight is above zero for every score but -inf, too small for fp32 or not)
                const float some = x == -INFINITY ? 0.0f : fmaxf(p, FLT_MIN);
#pragma unroll U
                for (int j = 0; j < lanes; ++j) {
                    const float pj = __shfl_sync(0xffffffffu, p, j * groups + group);
                    const float sj = __shfl_sync(0xffffffffu, some, j * groups + group);
                    float f[8];
                    unpack8<T>(values(r.v, j), f);
#pragma unroll
                    for (int c = 0; c < 8; ++c) acc[c] = fmaf(isinf(f[c]) ? sj : pj, f[c], acc[c]);
                }
            }
#pragma unroll
            for (int w = 16; w > 0; w >>= 1) l += __shfl_xor_sync(0xffffffffu, l, w);
#pragma unroll
            for (int c = 0; c < 8; ++c)
                for (int w = lanes; w < 32; w <<= 1) acc[c] += __shfl_xor_sync(0xffffffffu, acc[c], w);
        }
        const float inv = 1.0f / l;
        T* o = reinterpret_cast<T*>(result(i));
#pragma unroll
        for (int c = 0; c < 8; ++c) {
            if (group != 0) continue;
            if (is_nan >> c & 1u) o[c] = T(NAN);
            else if (left >> c & 1u) o[c] = l == 0.0f ? T(0.0f) : T(acc[c] * inv);
        }
    }
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
                    const float w = p0 + p < pieces ? top[row[k] * pieces + p0 + p] : -1.0f;
                    if (!(w < 0.0f)) {   // (a weight of zero too: an infinity behind it shows)
                        x[k].x = fmaf(w, v[k][p].x, x[k].x); x[k].y = fmaf(w, v[k][p].y, x[k].y);
                        x[k].z = fmaf(w, v[k][p].z, x[k].z); x[k].w = fmaf(w, v[k][p].w, x[k].w);
                    }
                }
        }
#pragma unroll
        for (int k = 0; k < K; ++k) {
            if (i0 + k * (int)blockDim.x >= all) continue;
            if ((!isfinite(x[k].x) || !isfinite(x[k].y) || !isfinite(x[k].z) || !isfinite(x[k].w)) &&
                !isnan(top[row[k] * pieces]))
                atomicOr(again, 1 << row[k]);
            const int tok = a.by_group(row0 + row[k]), head = kvh * a.group + row0 + row[k] - tok * a.group;
            *reinterpret_cast<uint2*>(a.out + 2 * (((int64_t)(q.begin + tok) * a.hq + head) * a.D + 4 * col[k])) =
                make_uint2(pack2<T>(x[k].x, x[k].y), pack2<T>(x[k].z, x[k].w));
        }
    }
}

// Joins (maximum, sum, row) pieces of up to 16 rows, which several warps or CTAs summed
// over different keys, in their order, and writes the rows out.  Whole block, 128 threads;
// behind it *again holds a bit per row for attn_rows_exact: some columns came out not finite,
// although the scores were (a row with a score that was not is NaN).
// stat(i, row, k) reads piece i's maximum (k = 0) or sum (1), value(i, row, c) its columns
// 4 c ... 4 c + 3; `share` holds 32 x pieces floats.  A piece with a score of NaN or +inf has
// a maximum of +inf (and no other has: a sum with it is NaN).  FAR: the pieces lie in memory,
// many of them maybe, and their reads' latency is what it costs (one token over 4,000, 31
// pieces: the call took 25 us with two at a time, 17 with eight; sixteen gave no more).
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
            // a row of no weight at all is zeros, one with a NaN sum NaN, whatever the values
            top[r * pieces + p] = l == 0.0f ? -1.0f : w * inv;
        }
        if (live && t == 0) {
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
