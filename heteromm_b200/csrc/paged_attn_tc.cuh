// paged_attn_tc.cuh — the tensor-core attention kernel's launcher.
#pragma once

#include "paged_attn.cuh"

namespace hmm {
namespace serve {

struct TcArgs {
    AttnArgs a;
    int min_rows;        // sequences of fewer rows are another kernel's
    int box_rows;        // rows of a TMA box: a power of two that divides page_tokens
    uint64_t wait_ns;    // limit of every bounded wait
};

// Whether the kernel can read this cache (head size, page size, strides).
bool chunk_applies(const AttnArgs& a);
// Rows of every sequence with at least min_rows rows (n_new * group).
hmm_status_t run_chunk(const AttnArgs& a, bool bf16, int min_rows, cudaStream_t st);

}  // namespace serve
}  // namespace hmm
