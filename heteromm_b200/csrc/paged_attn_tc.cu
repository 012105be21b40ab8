// paged_attn_tc.cu — page arrays as TMA tensors, and the chunk kernel over a cache of 16-bit
// values.
#include <cudaTypedefs.h>

#include <algorithm>
#include <mutex>

#include "paged_chunk.cuh"

namespace hmm {
namespace serve {
namespace {

PFN_cuTensorMapEncodeTiled_v12000 encode_fn() {
    static PFN_cuTensorMapEncodeTiled_v12000 fn = nullptr;
    static std::once_flag once;
    std::call_once(once, [] {
        void* p = nullptr;
        cudaDriverEntryPointQueryResult r;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &r) == cudaSuccess &&
            r == cudaDriverEntryPointSuccess)
            fn = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(p);
    });
    return fn;
}

// 16-bit values (or bytes) in boxes of 128 or 64 bytes of a row, swizzled over as many, zeros out of range.
hmm_status_t encode_map(CUtensorMap* m, void* base, int rank, const cuuint64_t* dims, const cuuint64_t* strides,
                        const cuuint32_t* box, bool bytes = false) {
    auto fn = encode_fn();
    if (!fn) return set_error(HMM_ERR_CUDA, "cuTensorMapEncodeTiled is unavailable");
    const cuuint32_t ones[4] = {1, 1, 1, 1};
    const CUresult r = fn(m, bytes ? CU_TENSOR_MAP_DATA_TYPE_UINT8 : CU_TENSOR_MAP_DATA_TYPE_UINT16, (cuuint32_t)rank,
                          base, dims, strides, box, ones, CU_TENSOR_MAP_INTERLEAVE_NONE,
                          bytes && box[0] == 64 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_128B,
                          CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return set_error(HMM_ERR_CUDA, "cuTensorMapEncodeTiled failed (%d)", (int)r);
    return HMM_OK;
}

}  // namespace

// Units: at most one more per sequence and head than its share of the tokens.
int64_t most_units(int64_t n_seq, int64_t n_tokens, int64_t group, int64_t hk, int64_t rows) {
    return (n_tokens * group / rows + n_seq) * hk;
}

// Whether the units can be too few for whole ones (the tokens' row blocks are as many at
// least, if no sequence is another kernel's).
bool may_split(int64_t n_tokens, int64_t group, int64_t hk, int64_t rows) {
    return (n_tokens * group + rows - 1) / rows * hk < device_sm_count();
}

hmm_status_t make_page_map(CUtensorMap* m, const AttnArgs& a, const Pages& p, int box_rows, bool codes) {
    const cuuint64_t dims[4] = {(cuuint64_t)a.D, (cuuint64_t)a.page_tokens, (cuuint64_t)a.hk, (cuuint64_t)a.n_pages};
    cuuint64_t strides[3] = {(cuuint64_t)p.token, (cuuint64_t)p.head, (cuuint64_t)p.page};
    for (int i = 0; i < 3; ++i)
        if (dims[i + 1] == 1) strides[i] = 16;   // never stepped over
    const cuuint32_t box[4] = {codes && a.D > 64 ? 128u : 64u, (cuuint32_t)box_rows, 1, 1};
    return encode_map(m, p.base, 4, dims, strides, box, codes);
}

hmm_status_t make_query_map(CUtensorMap* m, const AttnArgs& a, int box_heads, int box_tokens) {
    const cuuint64_t dims[3] = {(cuuint64_t)a.D, (cuuint64_t)a.hq, (cuuint64_t)a.b.n_tokens};
    const cuuint64_t strides[2] = {a.hq == 1 ? 16 : (cuuint64_t)a.q_head,
                                   a.b.n_tokens == 1 ? 16 : (cuuint64_t)a.q_token};
    const cuuint32_t box[3] = {64, (cuuint32_t)box_heads, (cuuint32_t)box_tokens};
    return encode_map(m, const_cast<unsigned char*>(a.q), 3, dims, strides, box);
}

bool chunk_applies(const AttnArgs& a) {
    return box_rows_of(a.page_tokens, TC_KEYS) >= 8;
}

size_t chunk_workspace(int64_t n_seq, int64_t n_tokens, int64_t n_heads, int64_t n_kv_heads, int64_t D, bool shared) {
    const int64_t group = std::max<int64_t>(1, n_heads / n_kv_heads), ctas = device_sm_count(), rows = unit_rows(D);
    size_t n = up256(4 * (size_t)most_units(n_seq, shared ? 2 * n_tokens : n_tokens, group, n_kv_heads, rows) *
                     TC_SOFTMAX_WARPS);
    if (shared || may_split(n_tokens, group, n_kv_heads, rows))
        n += up256(2 * sizeof(int4) * ctas) +
             sizeof(float) * 2 * ctas * rows * ((D <= 64 ? 64 : D <= 128 ? 128 : 256) + 2);
    return n;
}

template hmm_status_t run_chunk<CODEC_NONE>(const AttnArgs&, bool, int, bool, unsigned char*, cudaStream_t, ChunkJoin*);

}  // namespace serve
}  // namespace hmm
