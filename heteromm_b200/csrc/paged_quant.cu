// paged_quant.cu — a paged cache held in 8 bits: what its calls check, filling it (the
// kernel of paged_append.cuh), and reading tokens back as rows of 16 or 32 bits.
//
// paged_quant_read_kernel.  Bound by memory: 33 bytes are read and 64 written for 32 values
// (16-bit rows).  A warp takes runs of four rows, whose places its lanes look up at once, and
// goes through their 16-byte vectors of codes, a lane with four in flight: the codes become
// values in a dozen integer instructions per four, without a table.  16 sequences of up to 8,192
// tokens, 8 heads of 128, e4m3 to fp16: 97 us, 4.6 TB/s (two rows' vectors in flight 101).
#include <algorithm>

#include "paged_append.cuh"
#include "paged_attn.cuh"

namespace hmm {
namespace serve {

hmm_status_t check_quant(const hmm_paged_quant_t* cache, const hmm_paged_batch_t* batch, Batch* b, Pages* k, Pages* v,
                         QuantRows* rows) {
    HMM_REQUIRE(cache && batch, "null cache or batch");
    HMM_REQUIRE(cache->codes == HMM_DTYPE_E4M3 || cache->codes == HMM_DTYPE_I8,
                "codes must be HMM_DTYPE_E4M3 or HMM_DTYPE_I8, got %d", (int)cache->codes);
    HMM_REQUIRE(cache->D >= Q_GROUP && cache->D <= 256 && cache->D % Q_GROUP == 0,
                "D must be a multiple of 32 in [32, 256], got %lld", (long long)cache->D);
    const hmm_paged_cache_t dims = quant_dims(*cache);
    const hmm_status_t s = check_batch(&dims, batch, b, k, v);
    if (s != HMM_OK) return s;
    const int64_t per = cache->D / Q_GROUP, block = cache->page_tokens * (cache->D + per);
    HMM_REQUIRE(cache->page_tokens * per % 16 == 0,
                "page_tokens * D / 32 must be a multiple of 16, got pages of %lld tokens and D %lld",
                (long long)cache->page_tokens, (long long)cache->D);
    const int64_t st[4] = {cache->k_page, cache->k_head, cache->v_page, cache->v_head};
    for (int i = 0; i < 4; ++i) {
        HMM_REQUIRE(st[i] >= 0 && st[i] % 16 == 0 && st[i] < (int64_t(1) << 40),
                    "cache strides must be multiples of 16 bytes below 2^40, got %lld", (long long)st[i]);
        HMM_REQUIRE((i & 1 ? cache->n_kv_heads : cache->n_pages) <= 1 || st[i] >= block,
                    "a page and head takes %lld bytes, the stride is %lld", (long long)block, (long long)st[i]);
    }
    *k = Pages{(unsigned char*)cache->k, cache->k_page, cache->k_head, cache->D};
    *v = Pages{(unsigned char*)cache->v, cache->v_page, cache->v_head, cache->D};
    *rows = QuantRows{cache->page_tokens * cache->D, (int)per};
    return HMM_OK;
}

namespace {

constexpr int RD_THREADS = 256;
constexpr int RD_ROWS = 4;     // rows whose places a warp looks up at once
constexpr int RD_DEPTH = 4;    // vectors of codes that a lane has in flight

struct ReadArgs {
    Batch b;
    Pages pages[2];
    unsigned char* out[2];     // [n_rows][heads][D], contiguous
    QuantRows rows;
    int64_t max_kv;
    int n_pages, hk, D, page_tokens;
    FastDiv by_head;           // vectors of a head
    int32_t* status;
};

template <typename O, int C>
__global__ void __launch_bounds__(RD_THREADS) paged_quant_read_kernel(const __grid_constant__ ReadArgs a) {
    const int lane = threadIdx.x & 31, warps = gridDim.x * (RD_THREADS / 32);
    const int per_row = a.hk * a.D / 16, per_head = a.D / 16;   // vectors of a row's keys, of a head
    for (int64_t t0 = (int64_t)(blockIdx.x * (RD_THREADS / 32) + (threadIdx.x >> 5)) * RD_ROWS; t0 < a.b.n_tokens;
         t0 += (int64_t)warps * RD_ROWS) {
        // the place of row t0 + lane: the last sequence that begins at or before it
        int phys = -1, slot = 0;
        if (lane < RD_ROWS && t0 + lane < a.b.n_tokens) {
            const int t = (int)t0 + lane;
            int s = 0;
            for (int n = a.b.n_seq; n > 1;) {   // s < s + n
                const int half = n >> 1;
                if (__ldg(a.b.cu + s + half) <= t) {
                    s += half;
                    n -= half;
                } else {
                    n = half;
                }
            }
            const int begin = __ldg(a.b.cu + s), end = __ldg(a.b.cu + s + 1), kv = __ldg(a.b.kv_len + s);
            if (t < begin || t >= end) {
                // a row of no sequence, left as it is (or cu is not ascending)
                if (t >= __ldg(a.b.cu) && t < __ldg(a.b.cu + a.b.n_seq)) atomicOr(a.status, HMM_STATUS_BATCH_BOUNDS);
            } else {
                const int64_t p = (int64_t)kv - end + t;
                if (begin < 0 || end > a.b.n_tokens || kv < 0 || kv > a.max_kv || p < 0) {
                    atomicOr(a.status, HMM_STATUS_BATCH_BOUNDS);
                } else {
                    const int logical = (int)p / a.page_tokens;
                    slot = (int)p - logical * a.page_tokens;
                    phys = __ldg(a.b.table + (int64_t)s * a.b.pages_per_seq + logical);
                    if (phys < 0 || phys >= a.n_pages) {
                        phys = -1;
                        atomicOr(a.status, HMM_STATUS_PAGE_BOUNDS);
                    }
                }
            }
        }
        for (int r = 0; r < RD_ROWS; ++r) {
            const int page = __shfl_sync(0xffffffffu, phys, r), in = __shfl_sync(0xffffffffu, slot, r);
            if (page < 0) continue;
            const int64_t row = (t0 + r) * a.hk * a.D;
            for (int i0 = lane; i0 < 2 * per_row; i0 += 32 * RD_DEPTH) {
                uint4 w[RD_DEPTH];
                uint32_t s[RD_DEPTH];
#pragma unroll
                for (int d = 0; d < RD_DEPTH; ++d) {
                    const int i = i0 + 32 * d;
                    if (i >= 2 * per_row) continue;
                    const int kv = i >= per_row, x = i - (kv ? per_row : 0), h = a.by_head(x), c = x - h * per_head;
                    const Pages& p = a.pages[kv];
                    const unsigned char* block = p.base + page * p.page + h * p.head;
                    w[d] = __ldg(reinterpret_cast<const uint4*>(block + (int64_t)in * a.D) + c);
                    s[d] = __ldg(block + a.rows.scales + (int64_t)in * a.rows.per_token + (c >> 1));
                }
#pragma unroll
                for (int d = 0; d < RD_DEPTH; ++d) {
                    const int i = i0 + 32 * d;
                    if (i >= 2 * per_row) continue;
                    const int kv = i >= per_row, x = i - (kv ? per_row : 0);
                    store16<O, C>(reinterpret_cast<O*>(a.out[kv]) + row + 16 * x, w[d], s[d]);
                }
            }
        }
    }
}

template <typename O>
hmm_status_t launch_read(const ReadArgs& a, bool e4m3, cudaStream_t st) {
    const int64_t warps = ((int64_t)a.b.n_tokens + RD_ROWS - 1) / RD_ROWS;
    const int64_t blocks = (warps + RD_THREADS / 32 - 1) / (RD_THREADS / 32);
    const unsigned grid = (unsigned)std::min<int64_t>(blocks, (int64_t)device_sm_count() * (2048 / RD_THREADS));
    if (e4m3) paged_quant_read_kernel<O, CODEC_E4M3><<<grid, RD_THREADS, 0, st>>>(a);
    else paged_quant_read_kernel<O, CODEC_I8><<<grid, RD_THREADS, 0, st>>>(a);
    return check_launch("paged_quant_read_kernel");
}

template <typename T>
hmm_status_t run_append(const AppendArgs& a, bool e4m3, int mode, int vpl, cudaStream_t st) {
    if (e4m3) return vpl == 2 ? launch_append<T, 2, CODEC_E4M3>(a, mode, st) : launch_append<T, 1, CODEC_E4M3>(a, mode, st);
    return vpl == 2 ? launch_append<T, 2, CODEC_I8>(a, mode, st) : launch_append<T, 1, CODEC_I8>(a, mode, st);
}

}  // namespace
}  // namespace serve
}  // namespace hmm

using namespace hmm;
using namespace hmm::serve;

extern "C" hmm_status_t hmm_paged_quant_append(
    const hmm_paged_quant_t* cache, const hmm_paged_batch_t* batch, int dtype, const void* q, int64_t q_token,
    int64_t q_head, int64_t n_heads, const void* k, int64_t k_token, int64_t k_head, const void* v,
    int64_t v_token, int64_t v_head, const void* q_weight, const void* k_weight, int weight_dtype,
    float eps, const float* rope, int64_t n_pos, int64_t rotary_dim, int interleaved,
    const int32_t* positions, void* q_out, int64_t out_token, int64_t out_head,
    int32_t* device_status, void* stream) {
    AppendArgs a{};
    hmm_status_t s = check_quant(cache, batch, &a.b, &a.k_pages, &a.v_pages, &a.quant);
    if (s != HMM_OK) return s;
    HMM_REQUIRE(dtype == HMM_DTYPE_BF16 || dtype == HMM_DTYPE_F16,
                "dtype must be HMM_DTYPE_BF16 or HMM_DTYPE_F16, got %d", dtype);
    hmm_paged_cache_t dims = quant_dims(*cache);
    dims.dtype = dtype;
    int mode, vpl;
    s = plan_append({q, q_token, q_head, n_heads, k, k_token, k_head, v, v_token, v_head, q_weight, k_weight, weight_dtype,
                     eps, rope, n_pos, rotary_dim, interleaved, positions, q_out, out_token, out_head, device_status},
                    dims, batch, true, &a, &mode, &vpl);
    if (s != HMM_OK || vpl == 0) return s;
    const bool e4m3 = cache->codes == HMM_DTYPE_E4M3;
    return dtype == HMM_DTYPE_BF16 ? run_append<__nv_bfloat16>(a, e4m3, mode, vpl, (cudaStream_t)stream)
                                   : run_append<__half>(a, e4m3, mode, vpl, (cudaStream_t)stream);
}

extern "C" hmm_status_t hmm_paged_quant_read(const hmm_paged_quant_t* cache, const hmm_paged_batch_t* batch, int dtype,
                                             void* k_out, void* v_out, int32_t* device_status, void* stream) {
    ReadArgs a{};
    const hmm_status_t s = check_quant(cache, batch, &a.b, &a.pages[0], &a.pages[1], &a.rows);
    if (s != HMM_OK) return s;
    HMM_REQUIRE(dtype == HMM_DTYPE_BF16 || dtype == HMM_DTYPE_F16 || dtype == HMM_DTYPE_F32,
                "dtype must be HMM_DTYPE_BF16, HMM_DTYPE_F16 or HMM_DTYPE_F32, got %d", dtype);
    HMM_REQUIRE(device_status, "null device_status");
    if (batch->n_seq == 0 || batch->n_tokens == 0) return HMM_OK;
    HMM_REQUIRE(batch->pages_per_seq > 0, "tokens to read, but no pages in the page table");
    HMM_REQUIRE(k_out && v_out, "null k_out or v_out");
    HMM_REQUIRE(aligned16(k_out) && aligned16(v_out), "k_out and v_out must be 16-byte aligned");
    const size_t bytes = (size_t)batch->n_tokens * cache->n_kv_heads * cache->D * (dtype == HMM_DTYPE_F32 ? 4 : 2);
    const uintptr_t k0 = (uintptr_t)k_out, v0 = (uintptr_t)v_out;
    HMM_REQUIRE(k0 + bytes <= v0 || v0 + bytes <= k0, "k_out and v_out overlap");
    for (const Pages& p : a.pages) {
        const uintptr_t first = (uintptr_t)p.base;
        const uintptr_t end = first + (cache->n_pages > 0 ? (cache->n_pages - 1) * p.page : 0) +
                              (cache->n_kv_heads - 1) * p.head + a.rows.scales + cache->page_tokens * a.rows.per_token;
        HMM_REQUIRE(!p.base || ((k0 + bytes <= first || end <= k0) && (v0 + bytes <= first || end <= v0)),
                    "k_out or v_out overlaps the pages");
    }
    a.out[0] = (unsigned char*)k_out;
    a.out[1] = (unsigned char*)v_out;
    a.max_kv = batch->pages_per_seq * cache->page_tokens;
    a.n_pages = (int)cache->n_pages;
    a.hk = (int)cache->n_kv_heads;
    a.D = (int)cache->D;
    a.page_tokens = (int)cache->page_tokens;
    a.by_head = FastDiv::of(a.D / 16);
    a.status = device_status;
    const bool e4m3 = cache->codes == HMM_DTYPE_E4M3;
    const cudaStream_t st = (cudaStream_t)stream;
    return dtype == HMM_DTYPE_BF16  ? launch_read<__nv_bfloat16>(a, e4m3, st)
           : dtype == HMM_DTYPE_F16 ? launch_read<__half>(a, e4m3, st)
                                    : launch_read<float>(a, e4m3, st);
}
