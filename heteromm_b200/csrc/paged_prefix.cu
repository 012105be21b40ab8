// paged_prefix.cu — attention of a batch whose sequences share a prefix, group by group: the
// prefix's keys are gone through once with all of a group's rows.
//
//   with (l1, o1) the log of a row's sum of exponentials and its result over the prefix, and
//   (l2, o2) over the rest of its sequence,  l = log(e^l1 + e^l2),
//   o = e^(l1 - l) o1 + e^(l2 - l) o2
//
// A call of one batch becomes a batch of parts: for each group one whose rows are those of all
// its sequences (they lie one behind the other) and whose keys are the prefix, every one of
// them seen; and for each sequence one with the keys behind it.  paged_shared_kernel writes
// them down, the kernels of attention go through them as through sequences (a group's rows are
// many: the tensor-core kernel, cut over the CTAs; a decoding sequence's few: the rows kernel,
// both at once), each leaving (l, o) in fp32, and paged_merge_kernel joins the two.  So n
// sequences read a prefix once and not n times, and what it costs beside is 2 * 4 (D + 1)
// bytes a row written and read.
#include <algorithm>

#include "paged_attn.cuh"

namespace hmm {
namespace serve {
namespace {

constexpr int SH_THREADS = 1024;
constexpr int MG_THREADS = 256;

struct SharedArgs {
    Batch b;                     // the call's
    const int32_t* cu_group;     // [n_groups + 1] sequences
    const int32_t* prefix;       // [n_groups]
    int n_groups;
    int64_t max_kv;
    int4* parts;                 // [n_groups + n_seq][2]: of the groups, then of the sequences
    int32_t* of_group;           // [n_groups][3]: prefix in common, first sequence with rows, sequences with rows
    int32_t* status;
};

struct MergeArgs {
    AttnArgs a;                  // (part and lse null)
    const int4* parts;           // of the sequences
    const float* part;           // [2][n_tokens][hq][D]: behind the prefix, and over it
    const float* part_lse;       // [2][n_tokens][hq]
    float* lse;                  // or null
};

// The group of sequence s, or -1: the last that begins at or before it, if s is in it.
__device__ __forceinline__ int group_of(const SharedArgs& a, int s) {
    int g = 0;
    for (int n = a.n_groups; n > 1;) {   // in [g, g + n)
        const int half = n >> 1;
        if (__ldg(a.cu_group + g + half) <= s) {
            g += half;
            n -= half;
        } else {
            n = half;
        }
    }
    return a.n_groups > 0 && __ldg(a.cu_group + g) <= s && s < __ldg(a.cu_group + g + 1) ? g : -1;
}

// One block: groups and sequences are few beside the rows.
__global__ void __launch_bounds__(SH_THREADS) paged_shared_kernel(const __grid_constant__ SharedArgs a) {
    for (int g = threadIdx.x; g < a.n_groups; g += SH_THREADS) {
        const int begin = __ldg(a.cu_group + g), end = __ldg(a.cu_group + g + 1), n = __ldg(a.prefix + g);
        const bool ok = begin >= 0 && end >= begin && end <= a.b.n_seq && n >= 0 && n <= a.max_kv;
        if (!ok) atomicOr(a.status, HMM_STATUS_BATCH_BOUNDS);
        a.of_group[3 * g] = ok ? n : 0;
        a.of_group[3 * g + 1] = INT32_MAX;
        a.of_group[3 * g + 2] = 0;
    }
    __syncthreads();
    // a prefix ends where a sequence's new tokens begin, which are not shared
    for (int s = threadIdx.x; s < a.b.n_seq; s += SH_THREADS) {
        const Seq q = load_seq(a.b, a.max_kv, s, a.status);
        const int g = group_of(a, s);
        if (g < 0 || q.n_new == 0) continue;
        atomicMin(a.of_group + 3 * g, max(0, q.pos0));
        atomicMin(a.of_group + 3 * g + 1, s);
        atomicAdd(a.of_group + 3 * g + 2, 1);
    }
    __syncthreads();
    for (int g = threadIdx.x; g < a.n_groups; g += SH_THREADS) {
        // (one sequence alone has nothing to share)
        int n = __ldcg(a.of_group + 3 * g + 2) > 1 ? __ldcg(a.of_group + 3 * g) : 0, begin = 0, rows = 0;
        if (n > 0) {
            begin = __ldg(a.b.cu + __ldg(a.cu_group + g));
            rows = __ldg(a.b.cu + __ldg(a.cu_group + g + 1)) - begin;
            if (begin < 0 || rows < 0 || begin + (int64_t)rows > a.b.n_tokens) {
                atomicOr(a.status, HMM_STATUS_BATCH_BOUNDS);
                begin = rows = n = 0;
            }
        }
        // (positions behind every key: all of them are seen)
        a.parts[2 * g] = make_int4(begin, rows, n, INT32_MAX - 1 - rows);
        a.parts[2 * g + 1] = make_int4(0, n > 0 ? __ldcg(a.of_group + 3 * g + 1) : 0, a.b.n_tokens + begin, 0);
    }
    __syncthreads();
    for (int s = threadIdx.x; s < a.b.n_seq; s += SH_THREADS) {
        const Seq q = load_seq(a.b, a.max_kv, s, a.status);
        const int g = group_of(a, s);
        int n = 0;
        if (g >= 0 && q.n_new > 0) {   // (where cu_new descends its rows may not be the group's)
            const int4 all = __ldcg(a.parts + 2 * g);
            if (q.begin >= all.x && q.begin + q.n_new <= all.x + all.y) n = all.z;
        }
        int4* p = a.parts + 2 * ((int64_t)a.n_groups + s);
        p[0] = make_int4(q.begin, q.n_new, q.kv, q.pos0);
        p[1] = make_int4(n, s, q.begin, 0);
    }
}

// A warp per row.
template <typename T, int C>
__global__ void __launch_bounds__(MG_THREADS) paged_merge_kernel(const __grid_constant__ MergeArgs m) {
    asm volatile("griddepcontrol.wait;" ::: "memory");   // launched while the kernel before still runs
    const AttnArgs& a = m.a;
    const int lane = threadIdx.x & 31;
    const int64_t row = (int64_t)blockIdx.x * (MG_THREADS / 32) + (threadIdx.x >> 5), rows = (int64_t)a.b.n_tokens * a.hq;
    if (row >= rows) return;
    const int tok = (int)(row / a.hq), head = (int)(row - (int64_t)tok * a.hq);
    int s = warp_find_seq(a.b, tok);
    auto owns = [&](const int4& p) { return tok >= p.x && tok - p.x < p.y; };
    if (!owns(__ldcg(m.parts + 2 * (int64_t)s))) {
        // a row of no sequence, left as it is; or one that the search missed, which takes a cu_new
        // that ascends (another is flagged)
        if (!(__ldcg(a.status) & HMM_STATUS_BATCH_BOUNDS)) return;
        unsigned at = 0;
        for (int s0 = 0; at == 0 && s0 < a.b.n_seq; s0 += 32) {
            s = s0 + lane;
            at = __ballot_sync(0xffffffffu, s < a.b.n_seq && owns(__ldcg(m.parts + 2 * (int64_t)s)));
        }
        if (at == 0) return;
        s = __shfl_sync(0xffffffffu, s, __ffs(at) - 1);
    }
    const int4 p0 = __ldcg(m.parts + 2 * (int64_t)s), p1 = __ldcg(m.parts + 2 * (int64_t)s + 1);
    const int in = tok - p0.x;
    float l2 = __ldcg(m.part_lse + row), l1 = p1.x > 0 ? __ldcg(m.part_lse + rows + row) : -INFINITY;
    const float top = fmaxf(l1, l2), ref = top == -INFINITY ? 0.0f : top;
    float w1 = expf(l1 - ref), w2 = expf(l2 - ref);
    const float sum = w1 + w2;                           // (NaN if one is: so are the row and lse)
    w1 = sum == 0.0f ? 0.0f : w1 / sum;
    w2 = sum == 0.0f ? 0.0f : w2 / sum;
    if (lane == 0 && m.lse) m.lse[row] = sum == 0.0f ? -INFINITY : ref + logf(sum);
    bool fine = true;
    for (int c = lane; c < a.D / 4; c += 32) {
        const float4 y = __ldcg(reinterpret_cast<const float4*>(m.part + row * a.D) + c);
        float4 x = make_float4(w2 * y.x, w2 * y.y, w2 * y.z, w2 * y.w);
        if (p1.x > 0) {
            const float4 z = __ldcg(reinterpret_cast<const float4*>(m.part + (rows + row) * a.D) + c);
            x = make_float4(fmaf(w1, z.x, x.x), fmaf(w1, z.y, x.y), fmaf(w1, z.z, x.z), fmaf(w1, z.w, x.w));
        }
        fine = fine && isfinite(x.x) && isfinite(x.y) && isfinite(x.z) && isfinite(x.w);
        *reinterpret_cast<uint2*>(a.out + 2 * (row * a.D + 4 * c)) = make_uint2(pack2<T>(x.x, x.y), pack2<T>(x.z, x.w));
    }
    if (__all_sync(0xffffffffu, fine) || isnan(sum)) return;
    // Finite scores, but a column that is not: from the definition, over the sequence's own row
    // of the table.
    __syncwarp();
    const Seq q{p0.x, p0.y, p0.z, true, p0.w, 0, s, p0.x};
    const int kvh = head / a.group;
    attn_rows_exact<T, C, 1>(a, q, kvh, in * a.group + head - kvh * a.group, 1u);
}

// The parts of the workspace behind the attention's own.
struct PrefixSpace {
    size_t attention, parts, of_group, part, lse, all;
};
PrefixSpace prefix_space(int64_t n_seq, int64_t n_tokens, int64_t n_groups, int64_t n_heads, int64_t n_kv_heads, int64_t D,
                         bool quant, int64_t max_kv) {
    PrefixSpace w;
    w.attention = up256(quant ? quant_attention_workspace(n_seq + n_groups, n_tokens, n_heads, n_kv_heads, D, max_kv, 0, 0, true)
                              : attention_workspace(n_seq + n_groups, n_tokens, n_heads, n_kv_heads, D, true));
    w.parts = up256(2 * sizeof(int4) * (size_t)(n_seq + n_groups));
    w.of_group = up256(3 * sizeof(int32_t) * (size_t)n_groups);
    w.part = up256(2 * sizeof(float) * (size_t)(n_tokens * n_heads * D));
    w.lse = up256(2 * sizeof(float) * (size_t)(n_tokens * n_heads));
    w.all = w.attention + w.parts + w.of_group + w.part + w.lse;
    return w;
}

template <typename T, int C>
hmm_status_t run_prefix(AttnArgs a, const int32_t* cu_group, const int32_t* prefix, int64_t n_groups, const PrefixSpace& w,
                        unsigned char* ws, cudaStream_t st) {
    unsigned char* at = ws + w.attention;
    SharedArgs sh{a.b, cu_group, prefix, (int)n_groups, a.max_kv, (int4*)at, (int32_t*)(at + w.parts), a.status};
    at += w.parts + w.of_group;
    MergeArgs m{a, sh.parts + 2 * n_groups, (float*)at, (float*)(at + w.part), a.lse};
    m.a.lse = nullptr;
    hmm_status_t s = launch(paged_shared_kernel, dim3(1), SH_THREADS, 0, false, st, "paged_shared_kernel", sh);
    if (s != HMM_OK) return s;
    a.part = (float*)m.part;
    a.lse = (float*)m.part_lse;
    a.b.shared = sh.parts;
    a.b.n_seq += (int)n_groups;
    s = run_attention<T, C>(a, 0, ws, st);
    if (s != HMM_OK) return s;
    const int64_t rows = (int64_t)a.b.n_tokens * a.hq, blocks = (rows + MG_THREADS / 32 - 1) / (MG_THREADS / 32);
    HMM_REQUIRE(blocks < (int64_t(1) << 31), "n_tokens * n_heads is too large for one call");
    return launch(paged_merge_kernel<T, C>, dim3((unsigned)blocks), MG_THREADS, 0, true, st, "paged_merge_kernel", m);
}

// What both entry points check beside plan_attention.
hmm_status_t check_groups(const int32_t* cu_group, const int32_t* prefix, int64_t n_groups, int64_t n_seq) {
    HMM_REQUIRE(n_groups >= 0 && n_groups <= n_seq, "n_groups must be in [0, n_seq], got %lld", (long long)n_groups);
    HMM_REQUIRE(n_groups == 0 || (cu_group && prefix), "null cu_group or prefix_len");
    return HMM_OK;
}

}  // namespace
}  // namespace serve
}  // namespace hmm

using namespace hmm;
using namespace hmm::serve;

extern "C" size_t hmm_paged_prefix_attention_workspace_size(int64_t n_seq, int64_t n_tokens, int64_t n_groups,
                                                            int64_t n_heads, int64_t n_kv_heads, int64_t D) {
    if (n_seq < 0 || n_tokens < 0 || n_groups < 0 || n_heads < 1 || n_kv_heads < 1 || D < 1 || D > 256) return 0;
    return prefix_space(n_seq, n_tokens, n_groups, n_heads, n_kv_heads, D, false, 0).all;
}

extern "C" hmm_status_t hmm_paged_prefix_attention(const hmm_paged_cache_t* cache, const hmm_paged_batch_t* batch,
                                                   const int32_t* cu_group, const int32_t* prefix_len, int64_t n_groups,
                                                   const void* q, int64_t q_token, int64_t q_head, int64_t n_heads,
                                                   float scale, void* out, float* lse, int32_t* device_status,
                                                   void* workspace, size_t workspace_bytes, void* stream) {
    AttnArgs a{};
    hmm_status_t s = check_batch(cache, batch, &a.b, &a.k, &a.v);
    if (s == HMM_OK) s = check_groups(cu_group, prefix_len, n_groups, batch->n_seq);
    if (s != HMM_OK) return s;
    const size_t need = hmm_paged_prefix_attention_workspace_size(batch->n_seq, batch->n_tokens, n_groups, n_heads,
                                                                  cache->n_kv_heads, cache->D);
    bool nothing;
    s = plan_attention({q, q_token, q_head, n_heads, scale, 1, 0, 0, 0, out, lse, device_status, workspace, workspace_bytes,
                        need}, *cache, batch, false, &a, &nothing);
    if (s != HMM_OK || nothing) return s;
    const PrefixSpace w = prefix_space(batch->n_seq, batch->n_tokens, n_groups, n_heads, cache->n_kv_heads, cache->D,
                                       false, 0);
    return cache->dtype == HMM_DTYPE_BF16 ? run_prefix<__nv_bfloat16, CODEC_NONE>(a, cu_group, prefix_len, n_groups, w,
                                                                                  (unsigned char*)workspace, (cudaStream_t)stream)
                                          : run_prefix<__half, CODEC_NONE>(a, cu_group, prefix_len, n_groups, w,
                                                                           (unsigned char*)workspace, (cudaStream_t)stream);
}

extern "C" size_t hmm_paged_quant_prefix_attention_workspace_size(int64_t n_seq, int64_t n_tokens, int64_t n_groups,
                                                                  int64_t n_heads, int64_t n_kv_heads, int64_t D,
                                                                  int64_t max_kv) {
    if (n_seq < 0 || n_tokens < 0 || n_groups < 0 || n_heads < 1 || n_kv_heads < 1 || D < 1 || D > 256 || max_kv < 0) return 0;
    return prefix_space(n_seq, n_tokens, n_groups, n_heads, n_kv_heads, D, true, max_kv).all;
}

extern "C" hmm_status_t hmm_paged_quant_prefix_attention(const hmm_paged_quant_t* cache, const hmm_paged_batch_t* batch,
                                                         int dtype, const int32_t* cu_group, const int32_t* prefix_len,
                                                         int64_t n_groups, const void* q, int64_t q_token, int64_t q_head,
                                                         int64_t n_heads, float scale, void* out, float* lse,
                                                         int32_t* device_status, void* workspace, size_t workspace_bytes,
                                                         void* stream) {
    AttnArgs a{};
    hmm_status_t s = check_quant(cache, batch, &a.b, &a.k, &a.v, &a.quant);
    if (s != HMM_OK) return s;
    HMM_REQUIRE(dtype == HMM_DTYPE_BF16 || dtype == HMM_DTYPE_F16,
                "dtype must be HMM_DTYPE_BF16 or HMM_DTYPE_F16, got %d", dtype);
    s = check_groups(cu_group, prefix_len, n_groups, batch->n_seq);
    if (s != HMM_OK) return s;
    const int64_t max_kv = batch->pages_per_seq * cache->page_tokens;
    const size_t need = hmm_paged_quant_prefix_attention_workspace_size(batch->n_seq, batch->n_tokens, n_groups, n_heads,
                                                                        cache->n_kv_heads, cache->D, max_kv);
    bool nothing;
    s = plan_attention({q, q_token, q_head, n_heads, scale, 1, 0, 0, 0, out, lse, device_status, workspace, workspace_bytes,
                        need}, quant_dims(*cache), batch, true, &a, &nothing);
    if (s != HMM_OK || nothing) return s;
    const PrefixSpace w = prefix_space(batch->n_seq, batch->n_tokens, n_groups, n_heads, cache->n_kv_heads, cache->D,
                                       true, max_kv);
    unsigned char* ws = (unsigned char*)workspace;
    const cudaStream_t st = (cudaStream_t)stream;
    if (cache->codes == HMM_DTYPE_E4M3)
        return dtype == HMM_DTYPE_BF16
                   ? run_prefix<__nv_bfloat16, CODEC_E4M3>(a, cu_group, prefix_len, n_groups, w, ws, st)
                   : run_prefix<__half, CODEC_E4M3>(a, cu_group, prefix_len, n_groups, w, ws, st);
    return dtype == HMM_DTYPE_BF16 ? run_prefix<__nv_bfloat16, CODEC_I8>(a, cu_group, prefix_len, n_groups, w, ws, st)
                                   : run_prefix<__half, CODEC_I8>(a, cu_group, prefix_len, n_groups, w, ws, st);
}
