// paged_quant_attn.cu — attention of ragged chunks of new tokens over a paged cache held in 8
// bits: the entry point.
#include "paged_rows.cuh"

namespace hmm {
namespace serve {

template hmm_status_t run_attention<__nv_bfloat16, CODEC_E4M3>(const AttnArgs&, int, unsigned char*, cudaStream_t);
template hmm_status_t run_attention<__half, CODEC_E4M3>(const AttnArgs&, int, unsigned char*, cudaStream_t);
template hmm_status_t run_attention<__nv_bfloat16, CODEC_I8>(const AttnArgs&, int, unsigned char*, cudaStream_t);
template hmm_status_t run_attention<__half, CODEC_I8>(const AttnArgs&, int, unsigned char*, cudaStream_t);

}  // namespace serve
}  // namespace hmm

using namespace hmm;
using namespace hmm::serve;

extern "C" size_t hmm_paged_quant_attention_workspace_size(int64_t n_seq, int64_t n_tokens, int64_t n_heads,
                                                           int64_t n_kv_heads, int64_t D) {
    return hmm_paged_attention_workspace_size(n_seq, n_tokens, n_heads, n_kv_heads, D);
}

extern "C" hmm_status_t hmm_paged_quant_attention(const hmm_paged_quant_t* cache, const hmm_paged_batch_t* batch, int dtype,
                                                  const void* q, int64_t q_token, int64_t q_head, int64_t n_heads,
                                                  float scale, int causal, int64_t window, int64_t sinks, int64_t max_new,
                                                  void* out, float* lse, int32_t* device_status, void* workspace,
                                                  size_t workspace_bytes, void* stream) {
    AttnArgs a{};
    hmm_status_t s = check_quant(cache, batch, &a.b, &a.k, &a.v, &a.quant);
    if (s != HMM_OK) return s;
    HMM_REQUIRE(dtype == HMM_DTYPE_BF16 || dtype == HMM_DTYPE_F16,
                "dtype must be HMM_DTYPE_BF16 or HMM_DTYPE_F16, got %d", dtype);
    const size_t need = hmm_paged_quant_attention_workspace_size(batch->n_seq, batch->n_tokens, n_heads,
                                                                 cache->n_kv_heads, cache->D);
    bool nothing;
    s = plan_attention({q, q_token, q_head, n_heads, scale, causal, window, sinks, max_new, out, lse, device_status,
                        workspace, workspace_bytes, need}, quant_dims(*cache), batch, true, &a, &nothing);
    if (s != HMM_OK || nothing) return s;
    const int hint = (int)std::min<int64_t>(max_new, INT32_MAX);
    unsigned char* ws = (unsigned char*)workspace;
    const cudaStream_t st = (cudaStream_t)stream;
    if (cache->codes == HMM_DTYPE_E4M3)
        return dtype == HMM_DTYPE_BF16 ? run_attention<__nv_bfloat16, CODEC_E4M3>(a, hint, ws, st)
                                       : run_attention<__half, CODEC_E4M3>(a, hint, ws, st);
    return dtype == HMM_DTYPE_BF16 ? run_attention<__nv_bfloat16, CODEC_I8>(a, hint, ws, st)
                                   : run_attention<__half, CODEC_I8>(a, hint, ws, st);
}
