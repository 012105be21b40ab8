// paged_append.cu — the step before attention over a paged cache, in one pass:
// RMS norm of every query and key head, position rotation, and the store of
// keys and values into the cache's pages.
//
//   y = x / sqrt(mean(x^2) + eps) * w        (without a weight y = x)
//   (a, b) -> (a cos - b sin, b cos + a sin) on pairs of the first rotary_dim
//   values: neighbours (2i, 2i+1), or halves (i, i + rotary_dim / 2)
//
// The pass has to read and write every value once (2 B each way) and does a
// handful of fp32 operations on it, so HBM bounds it.  One CTA takes one token
// with all its heads: the token's sequence, page and angles are looked up once
// and the loads of its rows are issued before that lookup, so its latency (four
// dependent L2 reads) is hidden behind them.  A head's row lies in a group of
// 2^n lanes, 16 bytes a lane; the sum of squares is a butterfly in the group,
// the partner of a halves pair comes by a shuffle (its vector is rotary_dim/16
// lanes away), or through shared memory where rotary_dim/2 is no multiple of 8
// or a lane holds two vectors.  A lane's angles are the same for every head.  Everything is computed in fp32 and rounded once.
#include <algorithm>

#include "paged_serve.cuh"

namespace hmm {
namespace serve {

hmm_status_t check_batch(const hmm_paged_cache_t* cache, const hmm_paged_batch_t* batch, Batch* b,
                         Pages* k, Pages* v) {
    HMM_REQUIRE(cache && batch, "null cache or batch");
    HMM_REQUIRE(cache->dtype == HMM_DTYPE_BF16 || cache->dtype == HMM_DTYPE_F16,
                "dtype must be HMM_DTYPE_BF16 or HMM_DTYPE_F16, got %d", (int)cache->dtype);
    HMM_REQUIRE(cache->D >= 8 && cache->D <= 512 && cache->D % 8 == 0,
                "D must be a multiple of 8 in [8, 512], got %lld", (long long)cache->D);
    HMM_REQUIRE(cache->n_kv_heads >= 1 && cache->n_kv_heads <= 65535,
                "n_kv_heads must be in [1, 65535], got %lld", (long long)cache->n_kv_heads);
    HMM_REQUIRE(cache->page_tokens >= 1 && cache->page_tokens < (int64_t(1) << 31),
                "page_tokens must be >= 1");
    HMM_REQUIRE(cache->n_pages >= 0 && cache->n_pages < (int64_t(1) << 31),
                "n_pages must be in [0, 2^31)");
    HMM_REQUIRE(batch->n_seq >= 0 && batch->n_seq <= 65535, "n_seq must be in [0, 65535], got %lld",
                (long long)batch->n_seq);
    HMM_REQUIRE(batch->pages_per_seq >= 0 && batch->pages_per_seq < (int64_t(1) << 31),
                "pages_per_seq must be in [0, 2^31)");
    HMM_REQUIRE(batch->n_tokens >= 0 && batch->n_tokens < (int64_t(1) << 31),
                "n_tokens must be in [0, 2^31)");
    HMM_REQUIRE(batch->pages_per_seq * cache->page_tokens < (int64_t(1) << 31),
                "pages_per_seq * page_tokens must be < 2^31");
    if (batch->n_seq > 0 && batch->n_tokens > 0) {
        HMM_REQUIRE(batch->cu_new && batch->kv_len, "null cu_new or kv_len");
        HMM_REQUIRE(batch->page_table || batch->pages_per_seq == 0, "null page table");
        HMM_REQUIRE((cache->k && cache->v) || cache->n_pages == 0, "null page array");
    }
    const int64_t st[6] = {cache->k_page, cache->k_head, cache->k_token,
                           cache->v_page, cache->v_head, cache->v_token};
    for (int64_t s : st)
        HMM_REQUIRE(s >= 0 && s % 8 == 0,
                    "cache strides must be multiples of 8 elements, got %lld", (long long)s);
    HMM_REQUIRE(aligned16(cache->k) && aligned16(cache->v), "page arrays must be 16-byte aligned");
    b->table = batch->page_table;
    b->cu = batch->cu_new;
    b->kv_len = batch->kv_len;
    b->n_seq = (int)batch->n_seq;
    b->pages_per_seq = (int)batch->pages_per_seq;
    b->n_tokens = (int)batch->n_tokens;
    *k = Pages{(unsigned char*)cache->k, 2 * cache->k_page, 2 * cache->k_head, 2 * cache->k_token};
    *v = Pages{(unsigned char*)cache->v, 2 * cache->v_page, 2 * cache->v_head, 2 * cache->v_token};
    return HMM_OK;
}

namespace {

constexpr int AP_THREADS = 256;
constexpr int AP_UNROLL = 4;   // rows a lane group has in flight

enum RopeMode { ROPE_NONE, ROPE_PAIRS, ROPE_HALVES, ROPE_HALVES_SMEM };

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
    int lpr;                     // lanes of a row's group
    float eps;
    int32_t* status;
};

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

template <typename T>
__device__ __forceinline__ uint4 pack8(const float* f) {
    return make_uint4(pack2<T>(f[0], f[1]), pack2<T>(f[2], f[3]), pack2<T>(f[4], f[5]),
                      pack2<T>(f[6], f[7]));
}

template <typename T, int VPL, int MODE>
__global__ void __launch_bounds__(AP_THREADS) paged_append_kernel(const __grid_constant__ AppendArgs a) {
    extern __shared__ float sm[];             // ROPE_HALVES_SMEM: a row of D values per group
    __shared__ int sh_phys, sh_row, sh_pos;   // sh_pos -1: no such token
    const int t = blockIdx.x;
    const int lpr = a.lpr, group = threadIdx.x / lpr, gl = threadIdx.x % lpr;
    const int n_groups = blockDim.x / lpr;
    const int rows = a.hq + 2 * a.hk;
    float2 cs[VPL][8];   // (cos, sin) of each value's pair: the same for every row of the token

    for (int r0 = group; r0 < rows + group; r0 += AP_UNROLL * n_groups) {
        // every row's loads, before anything that depends on the token's place
        uint4 x[AP_UNROLL][VPL];
#pragma unroll
        for (int u = 0; u < AP_UNROLL; ++u) {
            const int r = r0 + u * n_groups;
            const bool is_q = r < a.hq, is_k = !is_q && r < a.hq + a.hk;
            const Rows& in = is_q ? a.q : is_k ? a.k : a.v;
            const int h = is_q ? r : is_k ? r - a.hq : r - a.hq - a.hk;
            const unsigned char* src = in.base + t * in.token + h * in.head;
#pragma unroll
            for (int j = 0; j < VPL; ++j) {
                const int vi = gl + j * lpr;
                x[u][j] = r < rows && vi < a.vecs ? *reinterpret_cast<const uint4*>(src + 16 * vi)
                                                  : make_uint4(0u, 0u, 0u, 0u);
            }
        }
        if (r0 == group) {
            if (threadIdx.x < 32) {
                const int s = warp_find_seq(a.b, t);
                if (threadIdx.x == 0) {
                    int phys = -1, row = 0, pos = -1;
                    const int begin = __ldg(a.b.cu + s), end = __ldg(a.b.cu + s + 1);
                    if (begin <= t && t < end) {
                        const int kv = __ldg(a.b.kv_len + s);
                        const int64_t p = (int64_t)kv - (end - begin) + (t - begin);
                        if (begin < 0 || end > a.b.n_tokens || kv < 0 || kv > a.max_kv || p < 0) {
                            atomicOr(a.status, HMM_STATUS_BATCH_BOUNDS);
                        } else {
                            const int e = __ldg(a.b.table + (int64_t)s * a.b.pages_per_seq +
                                                p / a.page_tokens);
                            const int64_t ap = a.positions ? (int64_t)__ldg(a.positions + t) : p;
                            if (e < 0 || e >= a.n_pages) {
                                atomicOr(a.status, HMM_STATUS_PAGE_BOUNDS);
                            } else if (MODE != ROPE_NONE && (ap < 0 || ap >= a.n_pos)) {
                                atomicOr(a.status, HMM_STATUS_BATCH_BOUNDS);
                            } else {
                                phys = e;
                                row = (int)(p % a.page_tokens);
                                pos = MODE == ROPE_NONE ? 0 : (int)ap;
                            }
                        }
                    } else if (t < __ldg(a.b.cu + a.b.n_seq) && t >= __ldg(a.b.cu)) {
                        atomicOr(a.status, HMM_STATUS_BATCH_BOUNDS);   // cu_new is not ascending
                    }
                    sh_phys = phys;
                    sh_row = row;
                    sh_pos = pos;
                }
            }
            __syncthreads();
            if (sh_pos < 0) return;   // a padding row, or one that was flagged: left as it is
            if (MODE != ROPE_NONE) {
                const float2* row = reinterpret_cast<const float2*>(a.rope) + (int64_t)sh_pos * a.half;
#pragma unroll
                for (int j = 0; j < VPL; ++j)
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        const int e = 8 * (gl + j * lpr) + i;
                        const int pair = MODE == ROPE_PAIRS ? e >> 1 : e < a.half ? e : e - a.half;
                        if (MODE != ROPE_PAIRS || (i & 1) == 0)
                            cs[j][i] = e < 2 * a.half ? __ldg(row + pair) : make_float2(1.0f, 0.0f);
                    }
            }
        }
#pragma unroll
        for (int u = 0; u < AP_UNROLL; ++u) {
            const int r = r0 + u * n_groups;
            const bool live = r < rows;
            const bool is_q = r < a.hq, is_k = !is_q && r < a.hq + a.hk;
            if (live && !is_q && !is_k) {   // a value head: stored as it is
                unsigned char* dst = a.v_pages.base + sh_phys * a.v_pages.page +
                                     (r - a.hq - a.hk) * a.v_pages.head + sh_row * a.v_pages.token;
#pragma unroll
                for (int j = 0; j < VPL; ++j) {
                    const int vi = gl + j * lpr;
                    if (vi < a.vecs) *reinterpret_cast<uint4*>(dst + 16 * vi) = x[u][j];
                }
            }
            // (a group past the last row, or on a value head, goes through the shuffles with its warp)
            float y[VPL][8];
            float ss = 0.0f;
#pragma unroll
            for (int j = 0; j < VPL; ++j) {
                unpack8<T>(x[u][j], y[j]);
#pragma unroll
                for (int i = 0; i < 8; ++i) ss = fmaf(y[j][i], y[j][i], ss);
            }
            const void* w = is_q ? a.w[0] : a.w[1];
            if (a.w[0] || a.w[1]) {
                for (int o = lpr >> 1; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
                if (w) {
                    const float inv = 1.0f / sqrtf(ss / (float)a.D + a.eps);
#pragma unroll
                    for (int j = 0; j < VPL; ++j) {
                        const int vi = gl + j * lpr;
                        if (vi >= a.vecs) continue;
                        float wf[8];
                        if (a.w_f32) {
                            const float4* p = reinterpret_cast<const float4*>(w) + 2 * vi;
                            const float4 lo = __ldg(p), hi = __ldg(p + 1);
                            wf[0] = lo.x; wf[1] = lo.y; wf[2] = lo.z; wf[3] = lo.w;
                            wf[4] = hi.x; wf[5] = hi.y; wf[6] = hi.z; wf[7] = hi.w;
                        } else {
                            unpack8<T>(__ldg(reinterpret_cast<const uint4*>(w) + vi), wf);
                        }
#pragma unroll
                        for (int i = 0; i < 8; ++i) y[j][i] = y[j][i] * inv * wf[i];
                    }
                }
            }
            if (MODE == ROPE_PAIRS) {
#pragma unroll
                for (int j = 0; j < VPL; ++j)
#pragma unroll
                    for (int i = 0; i < 8; i += 2) {
                        if (8 * (gl + j * lpr) + i >= 2 * a.half) continue;   // as it is, infinities too
                        const float p = y[j][i], q = y[j][i + 1];
                        y[j][i] = p * cs[j][i].x - q * cs[j][i].y;
                        y[j][i + 1] = q * cs[j][i].x + p * cs[j][i].y;
                    }
            } else if (MODE == ROPE_HALVES) {
                // vector gl holds values [8 gl, 8 gl + 8); half is a multiple of 8
                const int hv = a.half >> 3;
                const bool first = gl < hv, turned = gl < 2 * hv;
                const int partner = first ? gl + hv : turned ? gl - hv : gl;
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const float o = __shfl_sync(0xffffffffu, y[0][i], partner, lpr);
                    if (turned) y[0][i] = y[0][i] * cs[0][i].x + (first ? -o : o) * cs[0][i].y;
                }
            } else if (MODE == ROPE_HALVES_SMEM) {
                float* row = sm + group * a.D;
#pragma unroll
                for (int j = 0; j < VPL; ++j) {
                    const int vi = gl + j * lpr;
                    if (vi < a.vecs) {
#pragma unroll
                        for (int i = 0; i < 8; ++i) row[8 * vi + i] = y[j][i];
                    }
                }
                __syncwarp();
#pragma unroll
                for (int j = 0; j < VPL; ++j)
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        const int e = 8 * (gl + j * lpr) + i;
                        if (e >= 2 * a.half) continue;
                        const bool first = e < a.half;
                        const float o = row[first ? e + a.half : e - a.half];
                        y[j][i] = y[j][i] * cs[j][i].x + (first ? -o : o) * cs[j][i].y;
                    }
                __syncwarp();
            }
            if (live && (is_q || is_k)) {
                unsigned char* dst =
                    is_q ? a.out.base + t * a.out.token + r * a.out.head
                         : a.k_pages.base + sh_phys * a.k_pages.page +
                               (r - a.hq) * a.k_pages.head + sh_row * a.k_pages.token;
#pragma unroll
                for (int j = 0; j < VPL; ++j) {
                    const int vi = gl + j * lpr;
                    if (vi < a.vecs) *reinterpret_cast<uint4*>(dst + 16 * vi) = pack8<T>(y[j]);
                }
            }
        }
    }
}

template <typename T, int VPL>
hmm_status_t launch_append(const AppendArgs& a, int mode, int threads, cudaStream_t st) {
    const size_t smem = mode == ROPE_HALVES_SMEM ? sizeof(float) * (threads / a.lpr) * a.D : 0;
    const unsigned grid = (unsigned)a.b.n_tokens;
    switch (mode) {
        case ROPE_NONE: paged_append_kernel<T, VPL, ROPE_NONE><<<grid, threads, 0, st>>>(a); break;
        case ROPE_PAIRS: paged_append_kernel<T, VPL, ROPE_PAIRS><<<grid, threads, 0, st>>>(a); break;
        case ROPE_HALVES_SMEM:
            paged_append_kernel<T, VPL, ROPE_HALVES_SMEM><<<grid, threads, smem, st>>>(a);
            break;
        default: paged_append_kernel<T, 1, ROPE_HALVES><<<grid, threads, 0, st>>>(a); break;
    }
    return check_launch("paged_append_kernel");
}

}  // namespace
}  // namespace serve
}  // namespace hmm

using namespace hmm;
using namespace hmm::serve;

extern "C" hmm_status_t hmm_paged_kv_append(
    const hmm_paged_cache_t* cache, const hmm_paged_batch_t* batch, const void* q, int64_t q_token,
    int64_t q_head, int64_t n_heads, const void* k, int64_t k_token, int64_t k_head, const void* v,
    int64_t v_token, int64_t v_head, const void* q_weight, const void* k_weight, int weight_dtype,
    float eps, const float* rope, int64_t n_pos, int64_t rotary_dim, int interleaved,
    const int32_t* positions, void* q_out, int64_t out_token, int64_t out_head,
    int32_t* device_status, void* stream) {
    AppendArgs a{};
    hmm_status_t s = check_batch(cache, batch, &a.b, &a.k_pages, &a.v_pages);
    if (s != HMM_OK) return s;
    HMM_REQUIRE(n_heads >= 0 && n_heads <= 65535, "n_heads must be in [0, 65535], got %lld",
                (long long)n_heads);
    HMM_REQUIRE(device_status, "null device_status");
    HMM_REQUIRE(!rope || (rotary_dim >= 2 && rotary_dim % 2 == 0 && rotary_dim <= cache->D),
                "rotary_dim must be even and in [2, D], got %lld", (long long)rotary_dim);
    HMM_REQUIRE(!rope || (n_pos >= 0 && n_pos < (int64_t(1) << 31)), "n_pos out of range");
    HMM_REQUIRE(!(q_weight || k_weight) || weight_dtype == HMM_DTYPE_F32 || weight_dtype == cache->dtype,
                "norm weights must be fp32 or of the cache's type");
    HMM_REQUIRE(eps >= 0.0f, "eps must be >= 0");
    if (batch->n_seq == 0 || batch->n_tokens == 0) return HMM_OK;
    HMM_REQUIRE(batch->pages_per_seq > 0, "tokens to append, but no pages in the page table");
    HMM_REQUIRE(k && v && (n_heads == 0 || (q && q_out)), "null q, k, v or q_out");
    HMM_REQUIRE(aligned16(q) && aligned16(k) && aligned16(v) && aligned16(q_out) &&
                    aligned16(q_weight) && aligned16(k_weight) &&
                    (reinterpret_cast<uintptr_t>(rope) & 7) == 0,
                "q, k, v, q_out and the norm weights must be 16-byte aligned, rope 8-byte");
    const int64_t st[8] = {q_token, q_head, k_token, k_head, v_token, v_head, out_token, out_head};
    for (int64_t x : st)
        HMM_REQUIRE(x >= 0 && x % 8 == 0, "row strides must be multiples of 8 elements, got %lld",
                    (long long)x);
    a.q = Rows{(unsigned char*)const_cast<void*>(q), 2 * q_token, 2 * q_head};
    a.k = Rows{(unsigned char*)const_cast<void*>(k), 2 * k_token, 2 * k_head};
    a.v = Rows{(unsigned char*)const_cast<void*>(v), 2 * v_token, 2 * v_head};
    a.out = Rows{(unsigned char*)q_out, 2 * out_token, 2 * out_head};
    a.w[0] = q_weight;
    a.w[1] = k_weight;
    a.w_f32 = weight_dtype == HMM_DTYPE_F32;
    a.rope = rope;
    a.positions = positions;
    a.n_pos = n_pos;
    a.max_kv = batch->pages_per_seq * cache->page_tokens;
    a.n_pages = (int)cache->n_pages;
    a.hq = (int)n_heads;
    a.hk = (int)cache->n_kv_heads;
    a.D = (int)cache->D;
    a.vecs = a.D / 8;
    a.half = rope ? (int)(rotary_dim / 2) : 0;
    a.page_tokens = (int)cache->page_tokens;
    a.lpr = std::min(32, next_pow2(a.vecs));
    a.eps = eps;
    a.status = device_status;
    const int mode = !rope ? ROPE_NONE : interleaved ? ROPE_PAIRS
                     : a.half % 8 == 0 && a.vecs <= 32 ? ROPE_HALVES : ROPE_HALVES_SMEM;
    // as many lane groups as give each AP_UNROLL rows
    const int64_t groups = ((int64_t)a.hq + 2 * a.hk + AP_UNROLL - 1) / AP_UNROLL;
    const int threads = (int)std::min<int64_t>(AP_THREADS, (groups * a.lpr + 31) / 32 * 32);
    const cudaStream_t cs = (cudaStream_t)stream;
    if (cache->dtype == HMM_DTYPE_BF16)
        return a.vecs > 32 ? launch_append<__nv_bfloat16, 2>(a, mode, threads, cs)
                           : launch_append<__nv_bfloat16, 1>(a, mode, threads, cs);
    return a.vecs > 32 ? launch_append<__half, 2>(a, mode, threads, cs)
                       : launch_append<__half, 1>(a, mode, threads, cs);
}
