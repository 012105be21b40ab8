// paged_attn.cu — attention of ragged chunks of new tokens over a paged cache: the entry
// point.
#include "paged_rows.cuh"

namespace hmm {
namespace serve {

hmm_status_t plan_attention(const AttnCall& c, const hmm_paged_cache_t& dims, const hmm_paged_batch_t* batch, bool quant,
                            AttnArgs* args, bool* nothing) {
    const auto [q, q_token, q_head, n_heads, scale, causal, window, sinks, max_new, out, lse, device_status, workspace,
                workspace_bytes, need] = c;
    const hmm_paged_cache_t* cache = &dims;
    AttnArgs& a = *args;
    *nothing = true;
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
    *nothing = false;
    HMM_REQUIRE(cache->n_pages >= 1, "the cache has no pages");
    HMM_REQUIRE(batch->pages_per_seq * cache->page_tokens <= (int64_t(1) << 31) - 1024,
                "pages_per_seq * page_tokens must be <= 2^31 - 1024");   // ends of tiles stay in 31 bits
    if (!quant) {
        const int64_t steps[6] = {cache->page_tokens > 1 ? cache->k_token : 8, cache->n_kv_heads > 1 ? cache->k_head : 8,
                                  cache->n_pages > 1 ? cache->k_page : 8, cache->page_tokens > 1 ? cache->v_token : 8,
                                  cache->n_kv_heads > 1 ? cache->v_head : 8, cache->n_pages > 1 ? cache->v_page : 8};
        for (int64_t x : steps)
            HMM_REQUIRE(x > 0 && x < (int64_t(1) << 39), "cache strides must be in [8, 2^39) elements, got %lld",
                        (long long)x);
    }
    HMM_REQUIRE(q && out, "null q or out");
    HMM_REQUIRE(aligned16(q) && aligned16(out), "q and out must be 16-byte aligned");
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
    return HMM_OK;
}

size_t attention_workspace(int64_t n_seq, int64_t n_tokens, int64_t n_heads, int64_t n_kv_heads, int64_t D, bool shared) {
    // (the rows kernel over a cache in 8 bits has as many CTAs at least)
    return up256(rows_workspace<CODEC_E4M3>(rows_dp(D), shared)) + chunk_workspace(n_seq, n_tokens, n_heads, n_kv_heads, D, shared);
}

template <>
hmm_status_t run_attention<__nv_bfloat16, CODEC_NONE>(const AttnArgs& a, int max_new, unsigned char* ws, cudaStream_t st) {
    return run_kernels<__nv_bfloat16, CODEC_NONE>(a, max_new, ws, st);
}
template <>
hmm_status_t run_attention<__half, CODEC_NONE>(const AttnArgs& a, int max_new, unsigned char* ws, cudaStream_t st) {
    return run_kernels<__half, CODEC_NONE>(a, max_new, ws, st);
}

}  // namespace serve
}  // namespace hmm

using namespace hmm;
using namespace hmm::serve;

extern "C" size_t hmm_paged_attention_workspace_size(int64_t n_seq, int64_t n_tokens, int64_t n_heads,
                                                     int64_t n_kv_heads, int64_t D) {
    if (n_seq < 0 || n_tokens < 0 || n_heads < 1 || n_kv_heads < 1 || D < 1 || D > 256) return 0;
    return attention_workspace(n_seq, n_tokens, n_heads, n_kv_heads, D, false);
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
    bool nothing;
    const size_t need = hmm_paged_attention_workspace_size(batch->n_seq, batch->n_tokens, n_heads, cache->n_kv_heads,
                                                           cache->D);
    s = plan_attention({q, q_token, q_head, n_heads, scale, causal, window, sinks, max_new, out, lse, device_status,
                        workspace, workspace_bytes, need}, *cache, batch, false, &a, &nothing);
    if (s != HMM_OK || nothing) return s;
    const int hint = (int)std::min<int64_t>(max_new, INT32_MAX);
    return cache->dtype == HMM_DTYPE_BF16
               ? run_attention<__nv_bfloat16, CODEC_NONE>(a, hint, (unsigned char*)workspace, (cudaStream_t)stream)
               : run_attention<__half, CODEC_NONE>(a, hint, (unsigned char*)workspace, (cudaStream_t)stream);
}
