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

constexpr int TC_CTA_ROWS = 256;   // rows of a unit of the chunk kernel (D <= 128), at most

// What the join needs of units that the chunk kernel cut into pieces.
struct ChunkJoin {
    int4* joint;      // [ctas][2] unit begun in the CTA and ended in another: sequence, head, row block,
                      // pieces (0: none); the sequence's begin, n_new, kv
    float* part;      // [ctas][2][rows * (DP + 2)]: rows, then maxima, then sums
    int ctas, groups; // CTAs, 16-row groups of a unit that there can be
    int rows;         // of a unit
};

// Whether the kernel takes this page size: boxes of 8 rows and more.  Its producer's 32 lanes
// look up a tile's boxes, which boxes of 4 rows would just fit (not tried) and smaller ones
// not (2,048 tokens, 32/8 heads of 128: pages of 8 58 us here, of 4 837 in the rows kernel).
bool chunk_applies(const AttnArgs& a);
size_t chunk_workspace(int64_t n_seq, int64_t n_tokens, int64_t n_heads, int64_t n_kv_heads, int64_t D);
// Rows of every sequence with at least min_rows rows (n_new * group).  `behind`: the kernel
// before it on the stream is the rows kernel, which it may overlap and does not end before.
// *join says what is left to join (ctas = 0: nothing).
hmm_status_t run_chunk(const AttnArgs& a, bool bf16, int min_rows, bool behind, unsigned char* ws, cudaStream_t st,
                       ChunkJoin* join);

}  // namespace serve
}  // namespace hmm
