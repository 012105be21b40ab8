// paged_attn_tc.cuh — page arrays as TMA tensors, and the tensor-core attention
// kernel's launcher.
#pragma once

#include <cuda.h>

#include "paged_attn.cuh"
#include "sm100_ptx.cuh"

namespace hmm {
namespace serve {

// A page array as a tensor (D, page_tokens, heads, pages) of boxes {64, rows, 1, 1},
// 128-byte swizzle; values behind D and pages behind the last read as zeros.
hmm_status_t make_page_map(CUtensorMap* m, const AttnArgs& a, const Pages& p, int box_rows);

// Rows of a box: the largest power of two that divides page_tokens, at most `most`; a box
// never crosses a page's end.
inline int box_rows_of(int64_t page_tokens, int64_t most) {
    const int64_t r = page_tokens & -page_tokens;
    return (int)(r < most ? r : most);
}

// One box of a page array: values [x, x + 64) of rows y... of a head (z) and page (w).
__device__ __forceinline__ void tma_load_page(uint32_t dst, const CUtensorMap* map, uint64_t* bar, int x, int y,
                                              int z, int w) {
    asm volatile(
        "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes"
        " [%0], [%1, {%3, %4, %5, %6}], [%2];" ::"r"(dst),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(sm100::smem_u32(bar)), "r"(x), "r"(y), "r"(z), "r"(w)
        : "memory");
}

// Whether the kernel takes this head size and page size.
bool chunk_applies(const AttnArgs& a);
size_t chunk_workspace(int64_t n_seq, int64_t n_tokens, int64_t n_heads, int64_t n_kv_heads, int64_t D);
// Rows of every sequence with at least min_rows rows (n_new * group).  With more than one
// sequence the first word of ws must be 0 (the rows kernel, which runs before, sees to it).
hmm_status_t run_chunk(const AttnArgs& a, bool bf16, int min_rows, unsigned char* ws, cudaStream_t st);

}  // namespace serve
}  // namespace hmm
